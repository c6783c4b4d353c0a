// Attention of one query token per sequence over the paged key / value cache in 8 bits (format: kv8.cuh).
//
//   o[h] = sum_j p_j s_vj cv_j / sum_j p_j,   p_j = exp(scale s_kj (q[h] . ck_j) - max)
//
// for a key's codes ck, cv and scales s_k, s_v: the scales multiply scores and probabilities, so codes go to the tensor core as they are
// (e4m3 and int8 are subsets of f16) and a key costs its 2 (HD + 1) bytes and nothing else.
//
// * The products are S^T = K Q^T and O^T = V^T P^T (mma.sync): keys, then columns, are the 16 rows and eight query heads of one key head the columns.
//   Groups of up to eight heads, which is nearly all there are, fill the columns instead of half of 16 rows, and the accumulators of a head of
//   128 are 32 registers.  P^T reaches its operand layout by transposes of 8 x 8.
// * e4m3 and int8 are subsets of f16: codes are converted two at a time and multiplied by m16n8k16 with fp32 sums.  (m16n8k32 of e4m3 is made of
//   the same conversions and products on this GPU, and more of them.)  A query row is scaled by a power of two to a largest magnitude in [2^13,
//   2^14), exactly where its numbers are 2^-30 of that or more, and that power is taken out of its scores.  int8 has a product of its own for S^T,
//   m16n8k32 with int32 sums, without conversions: the query is 256 times one int8 number and another, the largest of a row in [2^14, 2^15).  Half a unit is
//   lost, so numbers below 2^-7 of the largest keep fewer bits than bf16 gave them, and a score moves by up to 2^-15 of the query's largest times the sum of the
//   key's magnitudes; rounding the key to int8 moved it by up to 2^-8 of the key's largest times the sum of the query's.
// * f16 does not hold every product p_j s_vj: every query head has a second reference, a power of two u with which its largest p_j s_vj so far is
//   between 2^7 and 2^15, and which rescales its accumulators like the reference of the scores does.  What f16 drops lies 2^-32 below that head's largest
//   product, whatever the scales of values are whose keys it does not look at.  (One power for all heads, taken from the scales alone, saves 3 % of
//   groups of 16 heads, 7 % of 8000 pairs of 30 keys and nothing of long sequences with up to eight heads, and loses everything 2^32 below the largest
//   scale, whether or not that has any weight.)
// * The contraction may take the columns of a head in any order, the output columns may lie anywhere, and so may the keys in the rows, so every
//   thread reads its operands as whole 16-byte pieces of a row and the exponents of its keys (four; two of a head of 256) as one word.  Rows are 128 bytes in shared memory
//   (half a row of a head of 256, two rows of a head of 64) in the 128-byte swizzle of the tensor-map copy; kv8_key says which key lies in
//   which row, so that the pieces that eight neighbouring lanes read lie in different banks, in both products.
// * Both references move only when a thread's p_j add up to more than 2^8 or a p_j s_vj u exceeds 2^15: a warp looks for that with one vote, where keeping the very maximum takes three
//   shuffles a column and a multiplication of all accumulators nearly every time.  The reference of scores is a whole number, so that both rescale by
//   powers of two, exactly.
// * Every warp has a ring of tiles of 32 keys (heads of 256: 16) of its own and waits for nobody while it streams; the sums of a CTA's four warps
//   meet in shared memory in the end.  (One ring for eight warps, fed by tensor-map copies: 130 clocks an SM for each of a tile's four copies, and
//   2 us at each end of a pair in which the SM's memory stood still.  CTAs that walk over equal parts of a list of all tiles: even, but nearly every
//   pair is cut, and a CTA that joins one or begins another stands still for 3 us.  128 x 1024 keys of 4 heads: 39 and 36 us, now 29.)
// * A CTA takes a chunk of a (sequence, key head) pair.  The lengths on the device decide how long chunks are, so that a captured launch serves any
//   of them: the smallest length that leaves no more chunks than the GPU holds CTAs, an even share where there are more pairs than that.  Chunks of a
//   cut pair leave their sums in the workspace, and the last one to finish, which a ticket of the pair tells, joins them.
//   Few pairs of up to 256 keys a warp get a cluster of up to 16 CTAs each, and the sums of the CTAs meet through distributed shared memory: no
//   ticket, no workspace.  Many short pairs get a warp each (zb_kv8_decode_plan).
// Bound by memory where sequences are long: one of 131072 keys, 8 key heads of 128, 50.5 us, 5.4 TB/s (82 % of a copy's rate; 38 us where the keys lie
// in L2); 128 of 1024 keys, 32 / 4 heads of 128, 29.1 us, 4.7 TB/s.  A launch has some 4.5 us that are not streaming: lengths, table and the first
// keys one after the other, and the sums at the end; sequences of unequal lengths that are not cut add the wait for the longest
// (32 of 128 - 2048 keys, 8 key heads of 128: 22.3 us, 3.3 TB/s).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "host_api.h"
#include "kv8.cuh"

namespace {

constexpr uint32_t kKernelKv8Decode = 41;
constexpr int kMaxBatch = 8192;                 // sequences whose lengths a CTA looks at: beyond, pairs are not cut
constexpr int kMinChunk = 8;                    // tiles: two for each warp
constexpr float kNoScore = -3.402823466e38f;    // the reference in front of the first key
constexpr float kMostP = 256.f;                 // what the p_j of a thread's keys may add up to before the references move
constexpr unsigned short kMostWeight = 0x7800;  // and p_j s_vj u grow to: 2^15 in f16
constexpr int kLift = 7;                        // log2 of what the largest p_j s_vj u is, at least, when they have moved
constexpr int kMostUnit = 237, kLeastUnit = 7;  // u is 2^-120 to 2^110, as exponent bytes: 1 / u, and p_j u, are numbers, too

struct Kv8DecodeParams {
  const __nv_bfloat16* q;
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const uint8_t* k_exps;
  const uint8_t* v_exps;
  __nv_bfloat16* out;
  const int32_t* block_table;
  const int32_t* seq_lens;
  float* part_o;               // [slots][rows][HD]: the sums of a cut pair's chunk
  float2* part_ml;             // [slots][rows]: reference and sum
  uint32_t* tickets;           // [pairs], zero between launches
  long long q_stride;
  int batch, hkv, group, blocks, rows;      // blocks: of `rows` query heads (the last one of fewer) in a group
  int page_size, max_pages, num_pages, window;
  int parts;                   // CTAs that the GPU holds; CLUSTER: CTAs of a cluster
  float scale_log2;
  ZbStatus* status;
};

ZB_DEVICE void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first product of a sum.
ZB_DEVICE void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
ZB_DEVICE void mma_int8_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
ZB_DEVICE void mma_int8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
ZB_DEVICE uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
ZB_DEVICE uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
ZB_DEVICE uint32_t lds16(uint32_t at) {
  uint32_t v;
  asm volatile("{.reg .b16 h; ld.shared.u16 h, [%1]; cvt.u32.u16 %0, h;}" : "=r"(v) : "r"(at) : "memory");
  return v;
}
ZB_DEVICE uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// Keys of a tile: two groups of eight rows of an operand's 16, twice that for heads of up to 128.
template <int HD>
constexpr int kv8_groups() { return HD == 256 ? 2 : 4; }

// Key of a tile in row `g` of the idx-th group of eight rows.  A thread's keys are neighbours, one word of exponents; in the low bits, rows
// g = 2 i and 2 i + 1 differ so that their pieces of S^T's operand lie in different halves of the banks, and rows g = 2 t (or 2 t + 1) over t
// so that eight lanes of O^T's operand meet eight banks.
template <int HD>
ZB_DEVICE int kv8_key(int g, int idx) {
  if constexpr (HD == 64) return 4 * ((g & 4) | ((((g >> 2) ^ g) & 1) << 1) | ((g >> 1) & 1)) + idx;
  else if constexpr (HD == 128) return 4 * (g ^ ((g >> 1) & 1)) + (idx ^ (2 * (g >> 2)));
  else return 2 * (((g & 1) << 2) | (((g ^ (g >> 1)) & 1) << 1) | (g >> 2)) + idx;
}
// What the idx-th key's offset in a swizzled tile differs from the first one's by.
template <int HD>
ZB_DEVICE constexpr uint32_t kv8_step(int idx) {
  return HD == 64 ? ((idx >> 1) * 144) ^ ((idx & 1) * 64) : idx * 144;
}
// Offset of 16-byte piece c of key r in a tile.
template <int HD>
ZB_DEVICE uint32_t kv8_at(int r, int c) {
  if constexpr (HD == 64) return (r >> 1) * 128 + (((((r & 1) << 2) + c) ^ ((r >> 1) & 7)) << 4);
  else return r * 128 + ((c ^ (r & 7)) << 4);
}
// The scale (its bits) of byte i of a word of exponents.
ZB_DEVICE uint32_t kv8_scale_of(uint32_t word, int i) { return (i < 3 ? word << (23 - 8 * i) : word >> 1) & 0x7f800000u; }
ZB_DEVICE uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
ZB_DEVICE uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
ZB_DEVICE void copy16(uint32_t to, const void* from, bool some) {      // zeros where not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(some ? 16u : 0u) : "memory");
}
ZB_DEVICE float2 load_peer2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
ZB_DEVICE float4 load_peer4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
ZB_DEVICE void store32(float* to, const float (&x)[8]) {      // on 32 bytes
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]),
               "f"(x[7])
               : "memory");
}
ZB_DEVICE void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
ZB_DEVICE void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Tiles of a sequence that its query sees, one where it sees none (the pair's output has to be written).
struct Kv8Span {
  int len, first, tile0, tiles;      // keys first .. len - 1, in tiles tile0 .. tile0 + tiles - 1
};
template <int kTile>
ZB_DEVICE Kv8Span kv8_span(const Kv8DecodeParams& p, int seq) {
  Kv8Span s;
  s.len = kv8_len(p.seq_lens, seq, p.max_pages * p.page_size);
  s.first = p.window > 0 ? max(0, s.len - p.window) : 0;
  s.tile0 = s.first / kTile;
  s.tiles = max(1, (s.len + kTile - 1) / kTile - s.tile0);
  return s;
}
// What a CTA does: tiles [begin, end) of a pair, chunk `nth` of `chunks`.
struct Kv8Work {
  Kv8Span span;
  int seq, pair;                     // pair of the sequence
  int begin, end, nth, chunks;
  int slot;                          // of the pair's first chunk, where there are several
};
ZB_DEVICE void kv8_cut(Kv8Work& w) {
  const int each = w.span.tiles / w.chunks, longer = w.span.tiles - each * w.chunks;
  w.begin = w.nth * each + min(w.nth, longer);
  w.end = w.begin + each + (w.nth < longer ? 1 : 0);
}
// false: there are fewer chunks.  `tiles`: shared memory for a number of each sequence.
template <int kTile>
ZB_DEVICE bool kv8_work(const Kv8DecodeParams& p, Kv8Work& w, int* tiles) {
  const int pairs = p.hkv * p.blocks;
  for (int s = threadIdx.x; s < p.batch; s += blockDim.x) tiles[s] = kv8_span<kTile>(p, s).tiles;
  __syncthreads();
  const int total = kv8_total(p.batch, [&](int s) { return tiles[s]; });
  int length = 0, chunks = 0;
  float each = 0.f;
  // tiles / length, rounded up: the product of the reciprocal is off by less than one, and corrected
  const auto chunks_of = [&](int s) {
    int n = static_cast<int>(static_cast<float>(tiles[s]) * each);
    n += n * length < tiles[s] ? 1 : 0;
    n += n * length < tiles[s] ? 1 : 0;
    return (n - 1) * length >= tiles[s] ? n - 1 : n;
  };
  const auto cut_by = [&](int n) {
    length = max(kMinChunk, n);
    each = 1.f / static_cast<float>(length);
    chunks = kv8_total(p.batch, chunks_of) * pairs;
  };
  if (p.batch * pairs > p.parts) {
    cut_by(static_cast<int>(static_cast<float>(total) * static_cast<float>(pairs) / static_cast<float>(p.parts)) + 1);
  } else {
    // Rounding up adds half a chunk a sequence on average, and less than a whole one: the length for the former if that fits, else for more
    const int room = p.parts / pairs;                  // chunks of all sequences, at least one each
    for (int more = 2 * p.batch; more <= 4 * p.batch; more += p.batch) {
      const int left = 4 * room - more;
      cut_by(left > 0 ? static_cast<int>(4.f * static_cast<float>(total) / static_cast<float>(left)) + 1 : total);
      if (chunks <= p.parts) break;
    }
  }
  const int at = blockIdx.x;
  if (at >= chunks) return false;
  int before;
  kv8_locate(p.batch, at, [&](int s) { return chunks_of(s) * pairs; }, w.seq, before);
  w.span = kv8_span<kTile>(p, w.seq);
  w.chunks = chunks_of(w.seq);
  w.pair = (at - before) / w.chunks;
  w.nth = (at - before) - w.pair * w.chunks;
  w.slot = 0;
  if (w.chunks > 1)
    w.slot = kv8_total(w.seq, [&](int s) {
      const int n = chunks_of(s);
      return n > 1 ? n * pairs : 0;
    }) + w.pair * w.chunks;
  kv8_cut(w);
  __syncthreads();                                     // the rings lie over the numbers
  return true;
}

// How pairs are shared out: chunks of them to CTAs (kChunks), each to a cluster of CTAs, or a CTA (kCluster), or each to a warp (kWarp).
enum Kv8Mode { kChunks, kCluster, kWarp };

template <int HD, int NB, Kv8Mode MODE>
struct Kv8Sizes {
  static constexpr int kGroups = kv8_groups<HD>(), kTile = 8 * kGroups;      // keys of a tile
  static constexpr int kTileBytes = kTile * HD;
  static constexpr int kStageBytes = 2 * kTileBytes;
  // A warp for each pair of heads of 64 has registers and shared memory for 15 on an SM, of three stages: 8000 pairs of 30 keys take 16.9 us, where 12 of
  // four stages take 19.1 and 8 of six 24.5
  static constexpr bool kMany = HD == 64 && NB == 1 && MODE == kWarp;
  static constexpr int kStages = HD == 64 && !kMany ? 6 : 3;
  static constexpr int kWarps = MODE == kWarp ? 1 : 4, kCtas = (kMany ? 15 : 8) / kWarps;      // of a CTA, and CTAs on an SM
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kPitch = HD + 4;                             // floats of a row of sums
  static constexpr int kSums = (kWarps / 2) * 8 * NB * kPitch;      // half of the warps leave theirs, the others add to them
  static constexpr int kSmem = kWarps * (kWarpBytes + kStages * 2 * kTile) + (kWarps + 1) * 8 * NB * 8 + 1024;
  static_assert(kSums * 4 <= kWarps * kWarpBytes, "the sums lie over the rings");
  static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

template <int HD, int NB, bool INT8, Kv8Mode MODE>
__global__ void __launch_bounds__(32 * Kv8Sizes<HD, NB, MODE>::kWarps, Kv8Sizes<HD, NB, MODE>::kCtas) zb_kv8_decode_kernel(const Kv8DecodeParams p) {
  using Z = Kv8Sizes<HD, NB, MODE>;
  constexpr int kStages = Z::kStages, kWarps = Z::kWarps, kTile = Z::kTile, kGroups = Z::kGroups, kMt = kGroups / 2, kRows = 8 * NB, kSteps = HD / 16;
  constexpr int kSubs = HD > 128 ? 2 : 1, kPieces = HD / 64;
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  zb_pdl_launch();
  zb_pdl_wait();
  uint8_t* const smem = smem_raw + ((1024u - (zb_smem_u32(smem_raw) & 1023u)) & 1023u);
  Kv8Work w;
  if constexpr (MODE != kChunks) {
    const int index = blockIdx.x / p.parts, pairs = p.hkv * p.blocks;
    w.seq = index / pairs;
    w.pair = index - w.seq * pairs;
    w.span = kv8_span<kTile>(p, w.seq);
    w.nth = blockIdx.x - index * p.parts;
    w.chunks = p.parts;
    w.slot = 0;
    kv8_cut(w);
  } else {
    if (!kv8_work<kTile>(p, w, reinterpret_cast<int*>(smem))) return;
  }
  const uint32_t smem_at = zb_smem_u32(smem), stages_at = smem_at + warp * Z::kWarpBytes;
  const uint32_t exps_at = smem_at + kWarps * Z::kWarpBytes + warp * kStages * 2 * kTile;
  float* const sums = reinterpret_cast<float*>(smem);  // [half of the warps][row][kPitch], over the rings
  float* const stats = reinterpret_cast<float*>(smem + kWarps * (Z::kWarpBytes + kStages * 2 * kTile));      // [warp, all][row][reference, sum]

  // copies run kStages - 1 tiles ahead
  const int kvh = w.pair / p.blocks, row0 = (w.pair - kvh * p.blocks) * kRows, rows = min(kRows, p.group - row0);
  const int32_t* const bt = p.block_table + static_cast<size_t>(w.seq) * p.max_pages;
  int f_tile = w.begin + warp, f_nth = 0, f_stage = 0, f_pages = 0;
  const int line = lane >> 3, in_line = lane & 7;      // a lane copies 16 bytes of each of four lines of 128 bytes
  const uint32_t copy_to = HD == 256 ? (line & 1) * kTile * 128 + (line >> 1) * 128 + ((in_line ^ (line >> 1)) << 4) : line * 128 + ((in_line ^ line) << 4);
  const auto fetch = [&]() {
    if (f_tile < w.end) {
      const int nth = f_nth & (32 / kMt - 1);
      if (nth == 0) {                                  // pages of the next 32 groups of 16 keys, one a lane
        const int tile = f_tile + (lane / kMt) * kWarps, key = (w.span.tile0 + tile) * kTile + (lane % kMt) * 16;
        const bool some = tile < w.end && key < w.span.len && key + 16 > w.span.first;
        f_pages = some ? bt[key / p.page_size] : 0;
        if (static_cast<uint32_t>(f_pages) >= static_cast<uint32_t>(p.num_pages)) {
          zb_record_error(p.status, ZB_ERR_BOUNDS, kKernelKv8Decode, 1u, static_cast<uint32_t>(f_pages));
          f_pages = 0;
        }
        // from here on: the row of the group's first key, in units of 16 rows
        f_pages = ((f_pages * p.hkv + kvh) * p.page_size + key % p.page_size) >> 4;
        if (!some) f_pages = -1;
      }
      const uint32_t to = stages_at + f_stage * Z::kStageBytes;
      constexpr int kCopies = 16 * HD / 512;
#pragma unroll
      for (int part = 0; part < kMt; ++part) {
        const int unit = __shfl_sync(0xffffffffu, f_pages, kMt * nth + part);
        const size_t from = static_cast<size_t>(max(unit, 0)) * (16 * HD) + lane * 16;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int n = part * kCopies + i;
          const uint32_t at = HD == 256 ? n * 256 + (copy_to ^ (((2 * n) & 7) << 4)) : n * 512 + (copy_to ^ ((n & 1) << 6));
          copy16(to + at, p.k_codes + from + i * 512, unit >= 0);
          copy16(to + Z::kTileBytes + at, p.v_codes + from + i * 512, unit >= 0);
        }
        if (lane < 2)                                  // exponents of the keys, of the values
          copy16(exps_at + f_stage * 2 * kTile + lane * kTile + part * 16, (lane ? p.v_exps : p.k_exps) + static_cast<size_t>(max(unit, 0)) * 16, unit >= 0);
      }
      if (++f_stage == kStages) f_stage = 0;
      ++f_nth;
      f_tile += kWarps;
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  const int g = lane >> 2, t4 = lane & 3;
  // what this thread reads of a stage: keys of row g in S^T = K Q^T, of rows 2 t4 and 2 t4 + 1 in O^T = V^T P^T, and the exponents of the former
  const uint32_t ex_off = kv8_key<HD>(g, 0) & ~(kGroups - 1);
  const uint32_t k_off = kv8_at<HD>(kv8_key<HD>(g, 0), t4);
  const uint32_t v_off0 = Z::kTileBytes + kv8_at<HD>(kv8_key<HD>(2 * t4, 0), HD == 64 ? g >> 1 : g) + (HD == 64 ? (g & 1) * 8 : 0);
  const uint32_t v_off1 = Z::kTileBytes + kv8_at<HD>(kv8_key<HD>(2 * t4 + 1, 0), HD == 64 ? g >> 1 : g) + (HD == 64 ? (g & 1) * 8 : 0);
  const uint32_t turn = HD == 128 && g >= 4 ? 0x1032 : 0x3210;     // kv8_key's order of the four
  int stage = 0;
  // queries (e4m3: f16, two registers for 16 columns; int8: both parts of 32 columns), and what a score has to be multiplied by (columns 2 t4,
  // 2 t4 + 1 of each block of eight)
  uint32_t qf[NB][kSteps][2];
  float factor[NB][2];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int r = b * 8 + g;
    const __nv_bfloat16* src = p.q + static_cast<size_t>(w.seq) * p.q_stride + static_cast<size_t>(kvh * p.group + row0 + min(r, rows - 1)) * HD;
    uint2 raw[kSteps];
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      raw[i] = *reinterpret_cast<const uint2*>(src + (t4 + 4 * (i >> 2)) * 16 + (i & 3) * 4);
      if (r >= rows) raw[i] = make_uint2(0u, 0u);
      const uint32_t x = raw[i].x & 0x7fff7fffu, y = raw[i].y & 0x7fff7fffu;
      top = max(max(top, max(x >> 16, x & 0xffffu)), max(y >> 16, y & 0xffffu));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(max((INT8 ? 268 : 267) - static_cast<int>(top >> 7), 1), 253);      // exponent of 2^14 or 2^13 over 2^floor(log2 top)
    const float up = __uint_as_float(static_cast<uint32_t>(e) << 23);
    const float down = __uint_as_float(top >= 0x7f80u ? 0x7fffffffu : static_cast<uint32_t>(254 - e) << 23);      // no numbers, no scores
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const float2 x = zb_unpack_bf16x2(raw[i].x), y = zb_unpack_bf16x2(raw[i].y);
      if constexpr (INT8) {
        const float f[4] = {x.x * up, x.y * up, y.x * up, y.y * up};
        uint32_t hi = 0u, lo = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = min(max(__float2int_rn(f[j]), -32639), 32639), h = (n + 128) >> 8;
          hi |= (static_cast<uint32_t>(h) & 255u) << (8 * j);
          lo |= (static_cast<uint32_t>(n) & 255u) << (8 * j);
        }
        qf[b][i & ~1][i & 1] = hi;
        qf[b][i | 1][i & 1] = lo;
      } else {
        qf[b][i][0] = pack_half2(x.x * up, x.y * up);
        qf[b][i][1] = pack_half2(y.x * up, y.y * up);
      }
    }
    factor[b][0] = __shfl_sync(0xffffffffu, down, 8 * t4) * p.scale_log2;
    factor[b][1] = __shfl_sync(0xffffffffu, down, 8 * t4 + 4) * p.scale_log2;
  }
  float o[NB][kSteps][4];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < kSteps; ++i) o[b][i][0] = o[b][i][1] = o[b][i][2] = o[b][i][3] = 0.f;
  float m[NB][2], l[NB][2];                       // references, and the sums of this thread's keys
#pragma unroll
  for (int b = 0; b < NB; ++b) m[b][0] = m[b][1] = kNoScore, l[b][0] = l[b][1] = 0.f;
  int unit[NB][2];                                // exponent bytes of u
#pragma unroll
  for (int b = 0; b < NB; ++b) unit[b][0] = unit[b][1] = kMostUnit;

  // A tile's work is S^T = K Q^T (products), the weights (weigh), and O^T += V^T P^T (multiply).  The last one runs beside the next tile's first:
  // neither waits for the other, and a tile's conversions fill the time of the other's products.  The tile's values wait in registers.
  constexpr int kWords = HD == 64 ? 2 : 4;
  uint32_t v[kSubs][kMt][4][kWords], pb[NB][kGroups];
  float s[NB][kMt][4];
#pragma unroll
  for (int i = 0; i < kSubs * kMt * 4 * kWords; ++i) v[i / (kMt * 4 * kWords)][(i / (4 * kWords)) % kMt][(i / kWords) & 3][i % kWords] = 0u;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < kGroups; ++i) pb[b][i] = 0u;

  const auto products = [&](uint32_t at) {
    const uint32_t k_at = at + k_off;
    int n[INT8 ? NB : 1][kMt][2][4];               // int8: the products of the two parts of a query
    float f[INT8 ? 1 : NB][kMt][2][4];             // e4m3: two sums, so that no product waits for the one before it
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      uint4 x[kGroups];                            // piece c of the keys
#pragma unroll
      for (int i = 0; i < kGroups; ++i) x[i] = lds128(((k_at ^ kv8_step<HD>(i)) ^ ((c & 1) << 6)) + (c >> 1) * kTile * 128);
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt) {
        const uint32_t y[4] = {x[2 * mt].x, x[2 * mt].y, x[2 * mt].z, x[2 * mt].w}, z[4] = {x[2 * mt + 1].x, x[2 * mt + 1].y, x[2 * mt + 1].z, x[2 * mt + 1].w};
        if constexpr (INT8) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int part = 0; part < 2; ++part) {
                const uint32_t b0 = qf[b][4 * c + 2 * h + part][0], b1 = qf[b][4 * c + 2 * h + part][1];
                if (c + h == 0) mma_int8_first(n[b][mt][part], y[2 * h], z[2 * h], y[2 * h + 1], z[2 * h + 1], b0, b1);
                else mma_int8(n[b][mt][part], y[2 * h], z[2 * h], y[2 * h + 1], z[2 * h + 1], b0, b1);
              }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            kv8_to_half<false>(y[i], a0, a2);
            kv8_to_half<false>(z[i], a1, a3);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              if (c == 0 && i < 2) mma_f16_first(f[b][mt][i], a0, a1, a2, a3, qf[b][i][0], qf[b][i][1]);
              else mma_f16(f[b][mt][i & 1], a0, a1, a2, a3, qf[b][4 * c + i][0], qf[b][4 * c + i][1]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4 * kMt; ++i) {
        if constexpr (INT8) s[b][i >> 2][i & 3] = fmaf(256.f, static_cast<float>(n[b][i >> 2][0][i & 3]), static_cast<float>(n[b][i >> 2][1][i & 3]));
        else s[b][i >> 2][i & 3] = f[b][i >> 2][0][i & 3] + f[b][i >> 2][1][i & 3];
      }
  };

  // values of half `mt` of the tile's keys, columns of half `sub` of a head of 256: keys of rows 2 t4, 2 t4 + 1, and the same eight rows further
  const auto read = [&](uint32_t at, int key0, int sub, int mt, uint32_t (&x)[4][kWords]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int idx = 2 * mt + (k >> 1);
      const uint32_t from = ((at + ((k & 1) ? v_off1 : v_off0)) ^ kv8_step<HD>(idx)) + sub * kTile * 128;
      if constexpr (HD == 64) {
        const uint2 y = lds64(from);
        x[k][0] = y.x, x[k][1] = y.y;
      } else {
        const uint4 y = lds128(from);
        x[k][0] = y.x, x[k][1] = y.y, x[k][2] = y.z, x[k][3] = y.w;
      }
      // codes of rows that nobody sees may be anything, e4m3's NaN, too
      const int key = key0 + kv8_key<HD>(2 * t4 + (k & 1), idx);
      if (key0 >= 0 && (key < w.span.first || key >= w.span.len)) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[k][i] = 0u;
      }
    }
  };
  const auto multiply = [&](int sub, int mt, const uint32_t (&x)[4][kWords]) {
    // columns of a word: pairs of keys of each
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      uint32_t a[4], c[4];
      kv8_to_half<INT8>(__byte_perm(x[0][i], x[1][i], 0x5140), a[0], a[1]);
      kv8_to_half<INT8>(__byte_perm(x[2][i], x[3][i], 0x5140), a[2], a[3]);
      kv8_to_half<INT8>(__byte_perm(x[0][i], x[1][i], 0x7362), c[0], c[1]);
      kv8_to_half<INT8>(__byte_perm(x[2][i], x[3][i], 0x7362), c[2], c[3]);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        mma_f16(o[b][sub * 8 + 2 * i], a[0], a[1], a[2], a[3], pb[b][2 * mt], pb[b][2 * mt + 1]);
        mma_f16(o[b][sub * 8 + 2 * i + 1], c[0], c[1], c[2], c[3], pb[b][2 * mt], pb[b][2 * mt + 1]);
      }
    }
  };
  const auto multiply_all = [&]() {
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt) multiply(sub, mt, v[sub][mt]);
  };

  // !WHOLE: some of the keys lie behind the end or in front of the window
  const auto weigh = [&](auto whole, bool first, uint32_t at, uint32_t ex, int key0) {
    constexpr bool WHOLE = decltype(whole)::value;
    uint32_t k_exps, v_exps;
    if constexpr (kGroups == 4) k_exps = __byte_perm(lds32(ex), 0u, turn), v_exps = __byte_perm(lds32(ex + kTile), 0u, turn);
    else k_exps = lds16(ex), v_exps = lds16(ex + kTile);
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt) read(at, WHOLE ? -1 : key0, sub, mt, v[sub][mt]);
    float vs[kGroups];                             // scales of the values; a row that is NaN has the byte 255, an infinity, and its codes of zero make a NaN of it
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int key = key0 + kv8_key<HD>(g, i);
      const bool see = WHOLE || (key >= w.span.first && key < w.span.len);
      vs[i] = see ? __uint_as_float(kv8_scale_of(v_exps, i)) : 0.f;
      const float ks = __uint_as_float(kv8_scale_of(k_exps, i));
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float& x = s[b][i >> 1][(i & 1) * 2];
        float& y = s[b][i >> 1][(i & 1) * 2 + 1];
        zb_unpack2(zb_mul2(zb_pack2(x, y), zb_mul2(zb_pack2(ks, ks), zb_pack2(factor[b][0], factor[b][1]))), x, y);
        if (!see) x = y = -INFINITY;
      }
    }
    // both columns' numbers go in packed pairs
    ZbF2 chance[NB][kGroups], sum[NB];
    uint32_t weight[NB][kGroups];
    bool moves = false;
    const auto chances = [&](int b) {              // p_j
      const ZbF2 less = zb_pack2(-m[b][0], -m[b][1]);
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        float x, y;
        zb_unpack2(zb_add2(zb_pack2(s[b][i >> 1][(i & 1) * 2], s[b][i >> 1][(i & 1) * 2 + 1]), less), x, y);
        chance[b][i] = zb_pack2(zb_ex2(x), zb_ex2(y));
        sum[b] = i == 0 ? chance[b][i] : zb_add2(sum[b], chance[b][i]);
      }
      float x, y;
      zb_unpack2(sum[b], x, y);
      moves = moves || x > kMostP || y > kMostP;
    };
    const auto weights = [&](int b) {              // p_j s_vj u
      const ZbF2 u = zb_pack2(__uint_as_float(static_cast<uint32_t>(unit[b][0]) << 23), __uint_as_float(static_cast<uint32_t>(unit[b][1]) << 23));
      __half2 most = __float2half2_rn(0.f);
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        float x, y;
        zb_unpack2(zb_mul2(zb_mul2(chance[b][i], u), zb_pack2(vs[i], vs[i])), x, y);
        weight[b][i] = pack_half2(x, y);
        most = __hmax2(most, *reinterpret_cast<const __half2*>(&weight[b][i]));
      }
      moves = moves || __hgt(__hmax(__low2half(most), __high2half(most)), __ushort_as_half(kMostWeight));
    };
    if (!first) {                                  // a warp's first tile has no references yet
#pragma unroll
      for (int b = 0; b < NB; ++b) chances(b), weights(b);
    }
    if (__any_sync(0xffffffffu, first || moves)) {
      int rise[NB][2], fall[NB][2];                // what both references rise by together, and 1 / u by
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < kGroups; ++i) mx = fmaxf(mx, s[b][i >> 1][(i & 1) * 2 + j]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(ceilf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16))), m[b][j]);
          rise[b][j] = static_cast<int>(fminf(mx - m[b][j], 512.f));         // whole; no number (no references yet, infinities): 0 or 512
          m[b][j] = mx;
        }
        chances(b);
        float top0 = 0.f, top1 = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
          const float scale = fminf(vs[i], __uint_as_float(253u << 23));
          float x, y;
          zb_unpack2(zb_mul2(chance[b][i], zb_pack2(scale, scale)), x, y);
          top0 = fmaxf(top0, x), top1 = fmaxf(top1, y);
        }
        uint32_t tops = __float_as_uint(top0) >> 23 | __float_as_uint(top1) >> 23 << 16;      // exponent bytes of this tile's largest p_j s_vj of both columns
        tops = __vmaxu2(tops, __shfl_xor_sync(0xffffffffu, tops, 4));
        tops = __vmaxu2(tops, __shfl_xor_sync(0xffffffffu, tops, 8));
        tops = __vmaxu2(tops, __shfl_xor_sync(0xffffffffu, tops, 16));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int lower = 254 + kLift - static_cast<int>(tops >> (16 * j) & 255u);      // with which this tile's largest is 2^7 to 2^8
          const int now = max(min(min(unit[b][j] + rise[b][j], lower), kMostUnit), kLeastUnit);
          fall[b][j] = unit[b][j] + rise[b][j] - now;
          unit[b][j] = now;
        }
        weights(b);
      }
      if (!first) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            l[b][j] *= __uint_as_float(static_cast<uint32_t>(max(127 - rise[b][j], 0)) << 23);
            const float shrink = __uint_as_float(static_cast<uint32_t>(max(127 - fall[b][j], 0)) << 23);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
              o[b][i][j] *= shrink;
              o[b][i][j + 2] *= shrink;
            }
          }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float x, y;
      zb_unpack2(sum[b], x, y);
      l[b][0] += x, l[b][1] += y;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) pb[b][i] = transpose8(weight[b][i]);
    }
  };

  for (int t = w.begin + warp; t < w.end; t += kWarps) {
    copies_wait<kStages - 2>();
    __syncwarp();                                  // everybody's copies of this tile have landed, and the last tile has been read
    fetch();
    const int key0 = (w.span.tile0 + t) * kTile;
    const uint32_t at = stages_at + stage * Z::kStageBytes, ex = exps_at + stage * 2 * kTile + ex_off;
    if (w.span.len > 0) {
      products(at);
      multiply_all();
      if (key0 >= w.span.first && key0 + kTile <= w.span.len) weigh(std::true_type(), t == w.begin + warp, at, ex, key0);
      else weigh(std::false_type(), t == w.begin + warp, at, ex, key0);
    }
    if (++stage == kStages) stage = 0;
  }
  multiply_all();

  // A thread's columns of a row are neighbours, eight of them (HD 64), or 16 of each 128.
  const auto column = [&](int i) { return HD == 64 ? g * 8 + 2 * i : (i >> 3) * 128 + g * 16 + 2 * (i & 7); };
  const int out_row = w.seq * p.hkv * p.group + kvh * p.group + row0;
  const auto put = [&](int r, int col, const float4& x, float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;    // a row that sees nothing is zero
    *reinterpret_cast<uint2*>(p.out + static_cast<size_t>(out_row + r) * HD + col) = make_uint2(zb_pack_bf16x2(x.x * inv, x.y * inv), zb_pack_bf16x2(x.z * inv, x.w * inv));
  };
  const auto one_over = [&](int b, int j) { return __uint_as_float(static_cast<uint32_t>(254 - unit[b][j]) << 23); };
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[b][j] += __shfl_xor_sync(0xffffffffu, l[b][j], 4);
      l[b][j] += __shfl_xor_sync(0xffffffffu, l[b][j], 8);
      l[b][j] += __shfl_xor_sync(0xffffffffu, l[b][j], 16);
    }
  if constexpr (MODE == kWarp) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = b * 8 + 2 * t4 + j;
        if (r >= rows) continue;
        const float by = one_over(b, j);
#pragma unroll
        for (int i = 0; i < kSteps; i += 2)
          put(r, column(i), make_float4(o[b][i][j] * by, o[b][i][j + 2] * by, o[b][i + 1][j] * by, o[b][i + 1][j + 2] * by), l[b][j]);
      }
    return;
  }
  // The CTA's sums: the warps' references, then half of the warps leave their sums, the others add theirs.
  constexpr int kPitch = Z::kPitch, kHalf = kWarps / 2, kFours = HD / 4;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (g == 0) *reinterpret_cast<float2*>(stats + (warp * kRows + b * 8 + 2 * t4 + j) * 2) = make_float2(m[b][j], l[b][j]);
  __syncthreads();
#pragma unroll
  for (int turns = 0; turns < 2; ++turns) {
    if ((warp >= kHalf) == (turns == 0)) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = b * 8 + 2 * t4 + j;
          if (r >= rows) continue;
          float top = kNoScore;
#pragma unroll
          for (int k = 0; k < kWarps; ++k) top = fmaxf(top, stats[(k * kRows + r) * 2]);
          const float by = zb_ex2(m[b][j] - top) * one_over(b, j);
#pragma unroll
          for (int i = 0; i < kSteps; i += 2) {
            float4* dst = reinterpret_cast<float4*>(sums + ((turns == 0 ? warp - kHalf : warp) * kRows + r) * kPitch + column(i));
            float4 x = make_float4(o[b][i][j] * by, o[b][i][j + 2] * by, o[b][i + 1][j] * by, o[b][i + 1][j + 2] * by);
            if (turns == 1) {
              const float4 y = *dst;
              x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            *dst = x;
          }
        }
    }
    __syncthreads();
  }
  // the CTA's sums of a row and four columns
  const auto sum_of = [&](int r, int col, float& top, float& sum) {
    top = kNoScore, sum = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) top = fmaxf(top, stats[(k * kRows + r) * 2]);
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const float2 st = *reinterpret_cast<const float2*>(stats + (k * kRows + r) * 2);
      sum += zb_ex2(st.x - top) * st.y;
    }
    float4 x = *reinterpret_cast<const float4*>(sums + r * kPitch + col);
#pragma unroll
    for (int k = 1; k < kHalf; ++k) {
      const float4 y = *reinterpret_cast<const float4*>(sums + (k * kRows + r) * kPitch + col);
      x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    return x;
  };
  if constexpr (MODE == kCluster) {
    const bool alone = w.chunks == 1;
    for (int i = threadIdx.x; i < rows * kFours; i += 32 * kWarps) {
      const int r = i / kFours, col = 4 * (i - r * kFours);
      float top, sum;
      const float4 x = sum_of(r, col, top, sum);
      if (alone) {
        put(r, col, x, sum);
      } else {
        *reinterpret_cast<float4*>(sums + r * kPitch + col) = x;
        if (col == 0) *reinterpret_cast<float2*>(stats + (kWarps * kRows + r) * 2) = make_float2(top, sum);
      }
    }
    if (alone) return;
    // those of the cluster's CTAs, each of which finishes a share of the columns
    __syncwarp();
    zb_cluster_arrive();
    zb_cluster_wait();
    const uint32_t sums_at = zb_smem_u32(sums), stats_at = zb_smem_u32(stats + kWarps * kRows * 2);
    for (int i = w.nth + p.parts * threadIdx.x; i < rows * kFours; i += p.parts * 32 * kWarps) {
      const int r = i / kFours, col = 4 * (i - r * kFours);
      float top = kNoScore, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c0 = 0; c0 < p.parts; c0 += 8) {
        float2 st[8];
        float4 x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c0 + c >= p.parts) continue;
          st[c] = load_peer2(zb_mapa(stats_at + r * 8, c0 + c));
          x[c] = load_peer4(zb_mapa(sums_at + (r * kPitch + col) * 4, c0 + c));
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c0 + c >= p.parts) continue;
          const float up = fmaxf(top, st[c].x), was = zb_ex2(top - up), by = zb_ex2(st[c].x - up);
          acc.x = acc.x * was + by * x[c].x, acc.y = acc.y * was + by * x[c].y, acc.z = acc.z * was + by * x[c].z, acc.w = acc.w * was + by * x[c].w;
          sum = sum * was + by * st[c].y;
          top = up;
        }
      }
      put(r, col, acc, sum);
    }
    __syncwarp();
    zb_cluster_arrive();                           // nobody leaves while another one reads its shared memory
    zb_cluster_wait();
    return;
  } else {
    const bool complete = w.chunks == 1;
    const auto slot_at = [&](int nth, int r) { return static_cast<size_t>(w.slot + nth) * p.rows + r; };
    for (int i = threadIdx.x; i < rows * kFours; i += 32 * kWarps) {
      const int r = i / kFours, col = 4 * (i - r * kFours);
      float top, sum;
      const float4 x = sum_of(r, col, top, sum);
      if (complete) {
        put(r, col, x, sum);
      } else {
        *reinterpret_cast<float4*>(p.part_o + slot_at(w.nth, r) * HD + col) = x;
        if (col == 0) p.part_ml[slot_at(w.nth, r)] = make_float2(top, sum);
      }
    }
    if (complete) return;
    __shared__ uint32_t drawn;
    __syncthreads();                               // all of the CTA's sums are written
    if (threadIdx.x == 0) {
      __threadfence();
      uint32_t* ticket = p.tickets + static_cast<size_t>(w.seq) * p.hkv * p.blocks + w.pair;
      drawn = atomicAdd(ticket, 1u);
      if (drawn == static_cast<uint32_t>(w.chunks - 1)) *ticket = 0u;      // for the next launch
      __threadfence();
    }
    __syncthreads();
    if (drawn != static_cast<uint32_t>(w.chunks - 1)) return;
    // a warp for each row: the weights of 32 chunks at a time, one a lane, and the sums of 16
    for (int r = warp; r < rows; r += kWarps) {
      float top = kNoScore, sum = 0.f;
      float acc[HD / 32];
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) acc[j] = 0.f;
      for (int i0 = 0; i0 < w.chunks; i0 += 32) {
        constexpr int kOnce = HD == 256 ? 8 : 16;
        const int most = min(32, w.chunks - i0);
        const float2 ml = lane < most ? __ldcg(&p.part_ml[slot_at(i0 + lane, r)]) : make_float2(kNoScore, 0.f);
        float x[kOnce][HD / 32];
        const auto load = [&](int i1) {
#pragma unroll
          for (int i = 0; i < kOnce; ++i)
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) x[i][j] = i1 + i < most ? __ldcg(p.part_o + slot_at(i0 + i1 + i, r) * HD + lane + 32 * j) : 0.f;
        };
        load(0);
        const float up = fmaxf(top, zb_warp_max(ml.x)), was = zb_ex2(top - up), f = zb_ex2(ml.x - up);
        top = up;
        sum = sum * was + zb_warp_sum(f * ml.y);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) acc[j] *= was;
        for (int i1 = 0; i1 < most; i1 += kOnce) {
          if (i1 > 0) load(i1);
#pragma unroll
          for (int i = 0; i < kOnce; ++i) {
            const float by = __shfl_sync(0xffffffffu, f, (i1 + i) & 31);
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) acc[j] += by * x[i][j];
          }
        }
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) p.out[static_cast<size_t>(out_row + r) * HD + lane + 32 * j] = __float2bfloat16(acc[j] * inv);
    }
  }
}

template <int HD, int NB, bool INT8, Kv8Mode MODE>
int launch_decode(const Kv8DecodeParams& p, int pairs, cudaStream_t stream) {
  using Z = Kv8Sizes<HD, NB, MODE>;
  const auto kernel = zb_kv8_decode_kernel<HD, NB, INT8, MODE>;
  static bool configured[16] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) return -21;
  cudaError_t e = cudaSuccess;
  if (!configured[dev]) {
    e = zb_config_smem(kernel, Z::kSmem);
    if (MODE == kCluster && e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);      // 16 CTAs
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[dev] = true;
  }
  if (MODE == kCluster) e = zb_launch_cluster(kernel, dim3(static_cast<unsigned>(pairs * p.parts)), dim3(32 * Z::kWarps), Z::kSmem, stream, p.parts, p);
  else if (MODE == kWarp) e = zb_launch(kernel, dim3(static_cast<unsigned>(pairs)), dim3(32), Z::kSmem, stream, p);
  else e = zb_launch(kernel, dim3(static_cast<unsigned>(pairs <= p.parts ? p.parts : pairs + p.parts)), dim3(32 * Z::kWarps), Z::kSmem, stream, p);
  zb_count_launch(1);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}
template <int HD, int NB, bool INT8>
int launch_decode(const Kv8DecodeParams& p, Kv8Mode mode, int pairs, cudaStream_t stream) {
  if (mode == kWarp) return launch_decode<HD, NB, INT8, kWarp>(p, pairs, stream);
  return mode == kCluster ? launch_decode<HD, NB, INT8, kCluster>(p, pairs, stream) : launch_decode<HD, NB, INT8, kChunks>(p, pairs, stream);
}
template <int HD, int NB>
int launch_decode(const Kv8DecodeParams& p, bool int8, Kv8Mode mode, int pairs, cudaStream_t stream) {
  return int8 ? launch_decode<HD, NB, true>(p, mode, pairs, stream) : launch_decode<HD, NB, false>(p, mode, pairs, stream);
}

// Chunks of cut pairs: at most as many as there are CTAs, or, where there are more pairs, two for each even share that such a pair has.
long long slots_of(int parts) { return 2ll * parts; }

// Query heads of a pair: 16 where the group has more than eight (a head of 256 has registers for eight).
int rows_of(int hd, int group) { return group > 8 && hd <= 128 ? 16 : 8; }
}  // namespace

extern "C" {

// How a call is cut: CTAs of a cluster as a negative number, 0 for a warp for each pair, or the CTAs that share the chunks, and (in *floats) the
// fp32 numbers of its workspace, which needs no particular contents.  max_len: keys of the longest sequence, or a bound of them; any number gives right results.
int zb_kv8_decode_plan(int batch, int hq, int hkv, int hd, int max_len, long long* floats) {
  *floats = 0;
  if (batch <= 0) return 0;
  if (hkv <= 0 || hq <= 0 || hq % hkv != 0 || (hd != 64 && hd != 128 && hd != 256)) return INT_MIN;
  ZbDeviceState* st = zb_device_state();
  if (!st) return INT_MIN;
  const int block = rows_of(hd, hq / hkv), blocks = (hq / hkv + block - 1) / block, rows = std::min(hq / hkv, block), warps = 4, tile = hd == 256 ? 16 : 32;
  const long long pairs = static_cast<long long>(batch) * hkv * blocks, longest = std::max(1, (max_len + tile - 1) / tile), tiles = pairs * longest;
  if (tiles > 0x3fffffffll) return INT_MIN;
  const int most = st->num_sms * 2;
  // CTAs for a pair: as many as give each warp a tile and fit on the GPU at once.  Of clusters of 16 only half as many fit, as each lies within a part of the
  // GPU (16 pairs of 8000 keys: 18.0 us in clusters of 16, 13.8 of eight)
  int size = 1;
  while (size < 16 && size * warps < longest && pairs * size * 2 <= (size == 8 ? most / 2 : most)) size *= 2;
  // Up to 256 keys a warp a cluster is better than chunks, which look at all lengths and join through memory (us, heads of 128, a cluster / chunks: 8 pairs of
  // 5000 and 10000 keys 8.7 / 10.4, 10.6 / 12.6, 64 of 4000 15.9 / 18.8, 128 of 1800 15.2 / 18.0), also where lengths differ (64 of
  // 500 - 4000 14.3 / 14.5; 16 of 300 - 8000 11.6 / 11.1); beyond, the longest sequence keeps the others waiting (64 of 100 - 8000 21.8 / 19.0)
  if (pairs * size <= most && longest * tile <= size * warps * 256) return -size;
  // More pairs than CTAs, none of them long: a warp for each, where a CTA for each takes a turn per 296 of them, most of it spent on getting
  // under way (us, heads of 128, a warp / a CTA: 512 pairs of 40, 300, 1000 keys 5.6 / 8.2, 13.7 / 16.4, 32.8 / 28.2, 1024 pairs of 1000 45.0 / 51.7,
  // 8000 of 30 30.9 / 97.7).  Up to 2048 keys, as a warp is alone with its pair: 4096 pairs of 1000, 2000, 4000 keys 162 / 166, 309 / 307, 604 / 591, but
  // eight of 1000, 2048, 4000 among 4088 of 100: 41 / 64, 61 / 66, 95 / 70
  if (batch > kMaxBatch || (pairs > most && longest * tile <= 2048 && longest * tile * most <= pairs * 300)) return 0;
  // Too many to cut: a CTA for each, which need not look at the other lengths.  Up to 2048 keys, as a CTA is alone with its pair: that is what one long
  // sequence costs among short ones, where of sequences of equal or evenly spread lengths chunks are 1 - 3 us slower at any length (us, heads of 128, 8 of
  // a sequence, a CTA / chunks: 32 sequences of 1000, 2000, 3000 keys 15.2 / 16.4, 25.0 / 26.4, 34.4 / 35.7, 128 - 2048 21.6 / 22.9, 200 - 3000 29.0 / 30.2;
  // one of 1000, 2048, 3000, 8000 among 31 of 100 9.6 / 9.4, 14.9 / 11.1, 20.5 / 11.5, 47.0 / 19.4, among 63 11.2 / 12.6, 16.4 / 14.0, 22.0 / 15.1, 49.4 / 17.7)
  if (2 * pairs > most && longest * tile <= 2048) return -1;
  const int parts = static_cast<int>(std::min<long long>(tiles, most));
  *floats = slots_of(parts) * rows * (hd + 2);
  return parts;
}

// The arguments of a call, as the caller packs them (ops/kv8.py).
struct ZbKv8Decode {
  const void* q;                                   // [batch, hq, hd], rows on 8 bytes
  const void *k_codes, *k_exps, *v_codes, *v_exps;  // contiguous, on 16 bytes
  void* out;                                       // [batch, hq, hd], contiguous, on 8 bytes
  const int32_t* block_table;
  const int32_t* seq_lens;
  float* work;                                     // the numbers that the plan asked for
  uint32_t* tickets;                               // [batch * hkv * blocks of queries] where the plan is chunks: zero before the call, and after it
  void* stream;
  long long q_stride;
  int batch, hq, hkv, hd, page_size, max_pages, num_pages, window, int8, parts;
  float scale;
};

int zb_kv8_decode(const ZbKv8Decode* c) {
  const int hq = c->hq, hkv = c->hkv, hd = c->hd, page_size = c->page_size;
  if (c->batch <= 0) return 0;
  if (hkv <= 0 || hq <= 0 || hq % hkv != 0 || (hd != 64 && hd != 128 && hd != 256)) return -30;
  if (page_size <= 0 || page_size % 16 != 0 || c->num_pages <= 0 || static_cast<long long>(c->num_pages) * hkv * page_size > 0x7fffffffll ||
      static_cast<long long>(c->max_pages) * page_size > 0x7fffff00ll)
    return -31;
  if (c->parts < -16 || c->parts > 65536) return -33;
  if (((reinterpret_cast<uintptr_t>(c->q) | reinterpret_cast<uintptr_t>(c->out)) & 7) != 0 || c->q_stride % 4 != 0) return -32;
  ZbDeviceState* st = zb_device_state();
  if (!st) return -20;
  const int block = rows_of(hd, hq / hkv);
  Kv8DecodeParams p = {};
  p.q = reinterpret_cast<const __nv_bfloat16*>(c->q);
  p.k_codes = reinterpret_cast<const uint8_t*>(c->k_codes);
  p.v_codes = reinterpret_cast<const uint8_t*>(c->v_codes);
  p.k_exps = reinterpret_cast<const uint8_t*>(c->k_exps);
  p.v_exps = reinterpret_cast<const uint8_t*>(c->v_exps);
  p.out = reinterpret_cast<__nv_bfloat16*>(c->out);
  p.block_table = c->block_table;
  p.seq_lens = c->seq_lens;
  p.batch = c->batch;
  p.hkv = hkv;
  p.group = hq / hkv;
  p.blocks = (p.group + block - 1) / block;
  p.rows = std::min(p.group, block);
  const long long pairs = static_cast<long long>(c->batch) * hkv * p.blocks;
  if (pairs > 0x3ffffff) return -34;
  const Kv8Mode mode = c->parts > 0 ? kChunks : c->parts < 0 ? kCluster : kWarp;
  p.parts = std::max({1, c->parts, -c->parts});
  p.part_o = c->work;
  p.tickets = c->tickets;
  if (mode == kChunks) {
    if (c->batch > kMaxBatch || c->work == nullptr || c->tickets == nullptr) return -33;
    p.part_ml = reinterpret_cast<float2*>(c->work + slots_of(c->parts) * p.rows * hd);
  }
  p.q_stride = c->q_stride;
  p.page_size = page_size;
  p.max_pages = c->max_pages;
  p.num_pages = c->num_pages;
  p.window = c->window;
  p.scale_log2 = c->scale * 1.4426950408889634f;
  p.status = st->status;
  if (pairs * std::max<long long>(1, (static_cast<long long>(c->max_pages) * page_size + 15) / 16) > 0x3fffffffll) return -34;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(c->stream);
  const int n = static_cast<int>(pairs);
  if (hd == 64) return block == 8 ? launch_decode<64, 1>(p, c->int8 != 0, mode, n, s) : launch_decode<64, 2>(p, c->int8 != 0, mode, n, s);
  if (hd == 128) return block == 8 ? launch_decode<128, 1>(p, c->int8 != 0, mode, n, s) : launch_decode<128, 2>(p, c->int8 != 0, mode, n, s);
  return launch_decode<256, 1>(p, c->int8 != 0, mode, n, s);
}

}  // extern "C"
