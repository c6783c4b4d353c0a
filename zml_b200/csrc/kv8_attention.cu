// Attention of one query token per sequence over the paged key / value cache in 8 bits (format: kv8.cuh).
//
//   o[h] = sum_j p_j s_vj cv_j / sum_j p_j,   p_j = exp(scale s_kj (q[h] . ck_j) - max)
//
// for a key's codes ck, cv and scales s_k, s_v: the scales multiply scores and probabilities, so codes go to the tensor core as they are
// (e4m3 and int8 are subsets of f16) and a key costs its 2 (HD + 1) bytes and nothing else.
//
// * The products are S^T = K Q^T and O^T = V^T P^T (mma.sync m16n8k16, f16 inputs, fp32 sums): 16 keys, then 16 columns, are the rows, and
//   eight query heads of one key head the columns.  Groups of up to eight heads, which is nearly all there are, fill the columns instead of
//   half of 16 rows, and the accumulators of a head of 128 are 32 registers.  P^T reaches its operand layout by two transposes of 8 x 8.
// * The contraction may take the columns of a head in any order and the output columns may lie anywhere, so every thread reads its operands as whole
//   16-byte pieces of a row.  Rows are 128 bytes in shared memory (half a row of a head of 256, two rows of a head of 64) in the 128-byte swizzle of
//   the tensor-map copy: the pieces that eight neighbouring lanes read lie in different banks.
// * f16 holds neither every bf16 query nor every product p_j s_vj.  A query row is scaled by a power of two to a largest magnitude in
//   [2^13, 2^14), exactly, and that power is taken out of its scores; s_vj is taken relative to the largest one so far, and the weight times
//   2^7: what f16 drops lies 2^-32 below.
// * The reference that scores are taken from, and that of the values' scales, move only when a score exceeds its reference by 2^8 or a scale its own:
//   the weights stay below 2^15, and a warp looks for that with one vote, where keeping the very maximum takes three shuffles a column
//   and a multiplication of all accumulators nearly every time.
// * All tiles of 64 keys of all (sequence, key head) pairs are one list, cut into equal parts, one for each CTA: whatever the mix of lengths,
//   all SMs stream alike.  A CTA whose part ends inside a pair leaves its sums in the workspace, and a second kernel joins each such
//   pair.  Lengths are read on the device, so a captured launch serves any of them; nothing outlives the two launches.
// * Four warps take 16 keys of a tile each; a fifth one feeds the ring of tiles, page numbers fetched 32 at a time.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "host_api.h"
#include "kv8.cuh"

int zb_make_tmap_u8_2d_ex(CUtensorMap* out, const void* base, long long rows, long long row_bytes, int box_bytes, int box_rows, int swizzle128);

namespace {

constexpr uint32_t kKernelKv8Decode = 41;
constexpr int kTile = 64;                       // keys
constexpr int kMaxCtas = 384;                   // of the partition: what the joining kernel keeps weights for
constexpr float kNoScore = -3.402823466e38f;    // the reference in front of the first key
constexpr float kSlack = 8.f;                   // in units of log2: how far a score may exceed its reference
constexpr uint32_t kLift = 7;                   // log2 of what weights are multiplied by

struct Kv8DecodeParams {
  const __nv_bfloat16* q;
  const uint8_t* k_exps;
  const uint8_t* v_exps;
  __nv_bfloat16* out;
  const int32_t* block_table;
  const int32_t* seq_lens;
  float* part_o;               // [2 * ctas][rows][HD]: a CTA's first and its last pair
  float2* part_ml;             // [2 * ctas][rows]: maximum and sum
  long long q_stride;
  int batch, hkv, group, blocks;      // blocks: of `rows` query heads in a group
  int page_size, max_pages, num_pages, window;
  int unit;                    // keys of one copy: the largest power of two up to 64 that divides a page
  int ctas;
  float scale_log2;
  ZbStatus* status;
};

ZB_DEVICE void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
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
ZB_DEVICE uint32_t lds8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
ZB_DEVICE uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
ZB_DEVICE uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
ZB_DEVICE void consumer_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Tiles of a sequence that its query sees, one where it sees none (the pair's output has to be written).
struct Kv8Span {
  int len, first, tile0, tiles;      // keys first .. len - 1, in tiles tile0 .. tile0 + tiles - 1
};
ZB_DEVICE Kv8Span kv8_span(const Kv8DecodeParams& p, int seq) {
  Kv8Span s;
  s.len = kv8_len(p.seq_lens, seq, p.max_pages * p.page_size);
  s.first = p.window > 0 ? max(0, s.len - p.window) : 0;
  s.tile0 = s.first / kTile;
  s.tiles = max(1, (s.len + kTile - 1) / kTile - s.tile0);
  return s;
}
// The list of `total` tiles in equal parts: part c begins at begin(c), the first ones are one longer.
struct Kv8Parts {
  int each, longer;
  ZB_DEVICE Kv8Parts(int total, int ctas) : each(total / ctas), longer(total - each * ctas) {}
  ZB_DEVICE int begin(int c) const { return c * each + min(c, longer); }
  ZB_DEVICE int of(int pos) const {                   // the part that holds a position
    const int turn = longer * (each + 1);
    return pos < turn ? pos / (each + 1) : longer + (pos - turn) / each;
  }
};

// A CTA's walk over its part: segments of one pair each.  Every warp walks on its own.
struct Kv8Walk {
  Kv8Span span;
  int seq, pair, begin, end;         // pair of the sequence, tiles [begin, end) of it
  int at, last;                      // positions in the list
};
ZB_DEVICE void kv8_segment(Kv8Walk& w) { w.end = min(w.span.tiles, w.begin + (w.last - w.at)); }
ZB_DEVICE bool kv8_start(const Kv8DecodeParams& p, Kv8Walk& w) {
  const int pairs = p.hkv * p.blocks;
  const auto count = [&](int s) { return kv8_span(p, s).tiles * pairs; };
  const int total = kv8_total(p.batch, count);
  const Kv8Parts parts(total, p.ctas);
  w.at = parts.begin(blockIdx.x);
  w.last = parts.begin(blockIdx.x + 1);
  if (w.at >= w.last) return false;
  int before;
  kv8_locate(p.batch, w.at, count, w.seq, before);
  w.span = kv8_span(p, w.seq);
  w.pair = (w.at - before) / w.span.tiles;
  w.begin = (w.at - before) - w.pair * w.span.tiles;
  kv8_segment(w);
  return true;
}
ZB_DEVICE bool kv8_next(const Kv8DecodeParams& p, Kv8Walk& w) {
  w.at += w.end - w.begin;
  if (w.at >= w.last) return false;
  w.begin = 0;
  if (++w.pair == p.hkv * p.blocks) {
    w.pair = 0;
    w.span = kv8_span(p, ++w.seq);
  }
  kv8_segment(w);
  return true;
}

template <int HD, int NB>
struct Kv8Sizes {
  static constexpr int kRows = 8 * NB;                              // query heads of a pair
  static constexpr int kTileBytes = kTile * HD;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = HD == 64 ? 9 : (HD == 128 ? (NB == 1 ? 5 : 4) : 5);
  static constexpr int kPitch = HD + 4;                             // floats of a row of the four warps' sums
  static constexpr int kExpBytes = kStages * 2 * kTile;
  static constexpr int kMergeBytes = 4 * kRows * kPitch * 4 + 4 * kRows * 3 * 4;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kExpBytes + kMergeBytes + 2 * kStages * 8 + 16;
  static constexpr int kPerSm = kSmem <= 113 * 1024 ? 2 : 1;
};

template <int HD, int NB, bool INT8>
__global__ void __launch_bounds__(160, Kv8Sizes<HD, NB>::kPerSm) zb_kv8_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                                                            const Kv8DecodeParams p) {
  using Z = Kv8Sizes<HD, NB>;
  constexpr int kStages = Z::kStages, kRows = Z::kRows, kSteps = HD / 16, kSubs = HD > 128 ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (zb_smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* exps = smem + kStages * Z::kStageBytes;                                // [stage][keys, values][64]
  float* sums = reinterpret_cast<float*>(exps + kStages * 2 * kTile);             // [warp][row][kPitch]
  float* stats = sums + 4 * kRows * Z::kPitch;                                    // [warp][row][maximum, sum, scale of the values]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(stats + 4 * kRows * 3);
  uint64_t* empty_bar = full_bar + kStages;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(empty_bar + kStages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      zb_mbar_init(&full_bar[s], 1);
      zb_mbar_init(&empty_bar[s], 4);
    }
    *abort_flag = 0u;
    zb_mbar_fence_init();
    zb_tma_prefetch_desc(&tmap_k);
    zb_tma_prefetch_desc(&tmap_v);
  }
  __syncthreads();
  zb_pdl_launch();
  zb_pdl_wait();
  Kv8Walk w;
  if (!kv8_start(p, w)) return;
  uint32_t stage = 0, phase = 0;
  bool dead = false;                                 // a wait ran out: the walk goes on without waiting, so that all meet at the barriers

  if (warp == 4) {
    const int per_tile = kTile / p.unit;
    do {
      const int kvh = w.pair / p.blocks;
      const int32_t* bt = p.block_table + static_cast<size_t>(w.seq) * p.max_pages;
      int pages = 0;                                 // of the 32 copies from a multiple of 32 on, one a lane
      int off = (w.span.tile0 + w.begin) * kTile % p.page_size;
      for (int t = w.begin; t < w.end; ++t) {
        if (((t - w.begin) * per_tile & 31) == 0) {
          const int key = (w.span.tile0 + t) * kTile + lane * p.unit;
          pages = key < w.span.len ? bt[key / p.page_size] : 0;
          if (static_cast<uint32_t>(pages) >= static_cast<uint32_t>(p.num_pages)) {
            if ((w.span.tile0 + w.end) * kTile > key) zb_record_error(p.status, ZB_ERR_BOUNDS, kKernelKv8Decode, 1u, static_cast<uint32_t>(pages));
            pages = 0;
          }
        }
        if (!dead) dead = !zb_mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag);
        dead = __any_sync(0xffffffffu, dead);
        const int key0 = (w.span.tile0 + t) * kTile;
        const int copies = min(per_tile, (max(w.span.len - key0, 0) + p.unit - 1) / p.unit);
        if (!dead && lane == 0) zb_mbar_expect_tx(&full_bar[stage], copies * p.unit * 2 * (HD + 1));
        uint8_t* ks = smem + stage * Z::kStageBytes;
        uint8_t* ex = exps + stage * 2 * kTile;
        for (int c = 0; c < copies; ++c) {
          const int page = __shfl_sync(0xffffffffu, pages, ((t - w.begin) * per_tile + c) & 31);
          const long long row = (static_cast<long long>(page) * p.hkv + kvh) * p.page_size + off;
          off += p.unit;
          if (off == p.page_size) off = 0;
          if (dead || lane != 0) continue;
          const int y = static_cast<int>(HD == 64 ? row >> 1 : row);
          uint8_t* to = ks + c * p.unit * (HD > 128 ? 128 : HD);
#pragma unroll
          for (int sub = 0; sub < kSubs; ++sub) {
            zb_tma_load_2d(to + sub * kTile * 128, &tmap_k, &full_bar[stage], sub * 128, y);
            zb_tma_load_2d(to + Z::kTileBytes + sub * kTile * 128, &tmap_v, &full_bar[stage], sub * 128, y);
          }
          zb_bulk_load(ex + c * p.unit, p.k_exps + row, p.unit, &full_bar[stage]);
          zb_bulk_load(ex + kTile + c * p.unit, p.v_exps + row, p.unit, &full_bar[stage]);
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    } while (kv8_next(p, w));
  } else {
    const int g = lane >> 2, t4 = lane & 3;
    // what this thread reads of a stage: keys g and g + 8 of the warp's 16 in S^T = K Q^T, values 2 t4, 2 t4 + 1 (and 8 further) in O^T = V^T P^T
    uint32_t k_off[2], v_off[4];
    if constexpr (HD == 64) {
      const int r = warp * 16 + g;
      k_off[0] = (r >> 1) * 128 + (((((r & 1) << 2) + t4) ^ ((r >> 1) & 7)) << 4);
      k_off[1] = (k_off[0] ^ 64u) + 512u;
      v_off[0] = Z::kTileBytes + (warp * 8 + t4) * 128 + (((g >> 1) ^ t4) << 4) + (g & 1) * 8;
      v_off[1] = v_off[0] ^ 64u;
      v_off[2] = v_off[1] + 512u;
      v_off[3] = v_off[0] + 512u;
    } else {
      const int r = warp * 16 + g, q = warp * 16 + 2 * t4;
      k_off[0] = r * 128 + (((2 * t4) ^ (r & 7)) << 4);
      k_off[1] = k_off[0] + 1024u;
      v_off[0] = Z::kTileBytes + q * 128 + ((g ^ (q & 7)) << 4);
      v_off[1] = Z::kTileBytes + (q + 1) * 128 + ((g ^ ((q + 1) & 7)) << 4);
      v_off[2] = v_off[0] + 1024u;
      v_off[3] = v_off[1] + 1024u;
    }
    const uint32_t stages_at = zb_smem_u32(smem), exps_at = zb_smem_u32(exps) + warp * 16 + g;
    bool first_segment = true;
    do {
      const int kvh = w.pair / p.blocks, row0 = (w.pair - kvh * p.blocks) * kRows, rows = min(kRows, p.group - row0);
      // queries, scaled to f16, and what a score has to be multiplied by (columns 2 t4, 2 t4 + 1 of each block of eight)
      uint32_t qf[NB][kSteps][2];
      float factor[NB][2];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int r = b * 8 + g;
        const __nv_bfloat16* src = p.q + static_cast<size_t>(w.seq) * p.q_stride + static_cast<size_t>(kvh * p.group + row0 + min(r, rows - 1)) * HD;
        uint2 raw[kSteps];
        uint32_t top = 0u;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          // 16-byte piece of the row that step s belongs to, and its four columns in there
          const int piece = HD == 64 ? t4 : (s >> 3) * 8 + 2 * t4 + ((s >> 2) & 1);
          raw[s] = *reinterpret_cast<const uint2*>(src + piece * 16 + (s & 3) * 4);
          if (r >= rows) raw[s] = make_uint2(0u, 0u);
          const uint32_t x = raw[s].x & 0x7fff7fffu, y = raw[s].y & 0x7fff7fffu;
          top = max(max(top, max(x >> 16, x & 0xffffu)), max(y >> 16, y & 0xffffu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max(267 - static_cast<int>(top >> 7), 1), 253);             // exponent of 2^13 / 2^floor(log2 top)
        const float up = __uint_as_float(static_cast<uint32_t>(e) << 23), down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const float2 x = zb_unpack_bf16x2(raw[s].x), y = zb_unpack_bf16x2(raw[s].y);
          qf[b][s][0] = pack_half2(x.x * up, x.y * up);
          qf[b][s][1] = pack_half2(y.x * up, y.y * up);
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
      uint32_t power = kLift + 1;                     // exponent byte that the values' scales are relative to
      float unit = __uint_as_float((254u + kLift - power) << 23);

      // 16 keys; !WHOLE: some of them lie behind the end or in front of the window
      const auto block = [&](auto whole, uint32_t at, uint32_t ex, int key0) {
        constexpr bool WHOLE = decltype(whole)::value;
        constexpr int kWords = HD == 64 ? 2 : 4;
        uint4 kx[2][kSteps / 4];
        uint32_t v[kSubs][4][kWords];
#pragma unroll
        for (int c = 0; c < kSteps / 4; ++c) {
          kx[0][c] = lds128(at + (c >> 1) * kTile * 128 + (k_off[0] ^ ((c & 1) << 4)));
          kx[1][c] = lds128(at + (c >> 1) * kTile * 128 + (k_off[1] ^ ((c & 1) << 4)));
        }
        const bool see0 = WHOLE || (key0 + g >= w.span.first && key0 + g < w.span.len);
        const bool see1 = WHOLE || (key0 + g + 8 >= w.span.first && key0 + g + 8 < w.span.len);
        const float ks0 = kv8_scale(lds8(ex)), ks1 = kv8_scale(lds8(ex + 8));
        uint32_t ve0 = lds8(ex + kTile), ve1 = lds8(ex + kTile + 8);
        if (!see0) ve0 = 0u;
        if (!see1) ve1 = 0u;
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (HD == 64) {
              const uint2 x = lds64(at + v_off[k]);
              v[sub][k][0] = x.x, v[sub][k][1] = x.y;
            } else {
              const uint4 x = lds128(at + sub * kTile * 128 + v_off[k]);
              v[sub][k][0] = x.x, v[sub][k][1] = x.y, v[sub][k][2] = x.z, v[sub][k][3] = x.w;
            }
            // codes of rows that nobody sees may be anything, e4m3's NaN, too
            const int key = key0 + 2 * t4 + (k & 1) + (k >> 1) * 8;
            if (!WHOLE && (key < w.span.first || key >= w.span.len)) {
#pragma unroll
              for (int i = 0; i < kWords; ++i) v[sub][k][i] = 0u;
            }
          }
        float s[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
#pragma unroll
        for (int c = 0; c < kSteps / 4; ++c) {
          const uint32_t wx[4] = {kx[0][c].x, kx[0][c].y, kx[0][c].z, kx[0][c].w}, wy[4] = {kx[1][c].x, kx[1][c].y, kx[1][c].z, kx[1][c].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            kv8_to_half<INT8>(wx[i], a0, a2);
            kv8_to_half<INT8>(wy[i], a1, a3);
#pragma unroll
            for (int b = 0; b < NB; ++b) mma_f16(s[b], a0, a1, a2, a3, qf[b][c * 4 + i][0], qf[b][c * 4 + i][1]);
          }
        }
        bool moves = max(ve0, ve1) > power;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[b][j] = see0 ? s[b][j] * (ks0 * factor[b][j]) : -INFINITY;
            s[b][j + 2] = see1 ? s[b][j + 2] * (ks1 * factor[b][j]) : -INFINITY;
            moves = moves || fmaxf(s[b][j], s[b][j + 2]) > m[b][j] + kSlack;
          }
        if (__any_sync(0xffffffffu, moves)) {
          // a row that is NaN has the byte 255: its scale stays an infinity, and its codes of zero make a NaN of it
          const uint32_t now = max(power, __reduce_max_sync(0xffffffffu, min(max(ve0, ve1), 253u)));
          const float shrink = now - power > 126u ? 0.f : __uint_as_float((127u - (now - power)) << 23);
          power = now;
          unit = __uint_as_float((254u + kLift - now) << 23);
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float mx = fmaxf(s[b][j], s[b][j + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)), m[b][j]);
              const float c = zb_ex2(m[b][j] - mx);
              m[b][j] = mx;
              l[b][j] *= c;
#pragma unroll
              for (int i = 0; i < kSteps; ++i) {
                o[b][i][j] *= c * shrink;
                o[b][i][j + 2] *= c * shrink;
              }
            }
        }
        const float vs0 = kv8_scale(ve0) * unit, vs1 = kv8_scale(ve1) * unit;
        uint32_t pb[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[b][j] = zb_ex2(s[b][j] - m[b][j]);
            s[b][j + 2] = zb_ex2(s[b][j + 2] - m[b][j]);
            l[b][j] += s[b][j] + s[b][j + 2];
          }
          pb[b][0] = transpose8(pack_half2(s[b][0] * vs0, s[b][1] * vs0));
          pb[b][1] = transpose8(pack_half2(s[b][2] * vs1, s[b][3] * vs1));
        }
        // columns of a word: pairs of keys of each
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            uint32_t a[4], c[4];
            kv8_to_half<INT8>(__byte_perm(v[sub][0][i], v[sub][1][i], 0x5140), a[0], a[1]);
            kv8_to_half<INT8>(__byte_perm(v[sub][2][i], v[sub][3][i], 0x5140), a[2], a[3]);
            kv8_to_half<INT8>(__byte_perm(v[sub][0][i], v[sub][1][i], 0x7362), c[0], c[1]);
            kv8_to_half<INT8>(__byte_perm(v[sub][2][i], v[sub][3][i], 0x7362), c[2], c[3]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              mma_f16(o[b][sub * 8 + 2 * i], a[0], a[1], a[2], a[3], pb[b][0], pb[b][1]);
              mma_f16(o[b][sub * 8 + 2 * i + 1], c[0], c[1], c[2], c[3], pb[b][0], pb[b][1]);
            }
          }
      };

      for (int t = w.begin; t < w.end; ++t) {
        if (!dead) dead = !zb_mbar_wait(&full_bar[stage], phase, abort_flag);
        dead = __any_sync(0xffffffffu, dead);
        const int key0 = (w.span.tile0 + t) * kTile + warp * 16;
        if (!dead && key0 < w.span.len && key0 + 16 > w.span.first) {
          const uint32_t at = stages_at + stage * Z::kStageBytes, ex = exps_at + stage * 2 * kTile;
          if (key0 >= w.span.first && key0 + 16 <= w.span.len) block(std::true_type(), at, ex, key0);
          else block(std::false_type(), at, ex, key0);
        }
        __syncwarp();
        if (lane == 0) zb_mbar_arrive(&empty_bar[stage]);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }

      // the four warps' sums of this segment
      const float power_of = __uint_as_float((power - kLift) << 23);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = l[b][j];
          x += __shfl_xor_sync(0xffffffffu, x, 4);
          x += __shfl_xor_sync(0xffffffffu, x, 8);
          x += __shfl_xor_sync(0xffffffffu, x, 16);
          const int r = b * 8 + 2 * t4 + j;
          if (g == 0) {
            float* st = stats + (warp * kRows + r) * 3;
            st[0] = m[b][j];
            st[1] = x;
            st[2] = power_of;
          }
          float* dst = sums + (warp * kRows + r) * Z::kPitch;
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const int col = HD == 64 ? g * 8 + 2 * i : (i >> 3) * 128 + g * 16 + 2 * (i & 7);
            *reinterpret_cast<float2*>(dst + col) = make_float2(o[b][i][j], o[b][i][j + 2]);
          }
        }
      }
      consumer_barrier();
      const bool complete = w.begin == 0 && w.end == w.span.tiles;
      const int slot = 2 * static_cast<int>(blockIdx.x) + (first_segment ? 0 : 1);
      for (int i = threadIdx.x; i < rows * (HD / 2); i += 128) {
        const int r = i / (HD / 2), col = 2 * (i - r * (HD / 2));
        float top = kNoScore;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, stats[(k * kRows + r) * 3]);
        float ax = 0.f, ay = 0.f, sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float* st = stats + (k * kRows + r) * 3;
          const float f = zb_ex2(st[0] - top), fo = f * st[2];
          const float2 x = *reinterpret_cast<const float2*>(sums + (k * kRows + r) * Z::kPitch + col);
          ax += fo * x.x;
          ay += fo * x.y;
          sum += f * st[1];
        }
        if (complete) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;            // a row that sees nothing is zero
          *reinterpret_cast<uint32_t*>(p.out + (static_cast<size_t>(w.seq) * p.hkv * p.group + kvh * p.group + row0 + r) * HD + col) =
              zb_pack_bf16x2(ax * inv, ay * inv);
        } else {
          *reinterpret_cast<float2*>(p.part_o + (static_cast<size_t>(slot) * kRows + r) * HD + col) = make_float2(ax, ay);
          if (col == 0) p.part_ml[static_cast<size_t>(slot) * kRows + r] = make_float2(top, sum);
        }
      }
      consumer_barrier();                             // the sums may be overwritten
      first_segment = false;
    } while (kv8_next(p, w));
  }
  __syncthreads();
  if (*abort_flag != 0u) {
    if (threadIdx.x == 0) zb_record_error(p.status, ZB_ERR_MBAR_TIMEOUT, kKernelKv8Decode, 1u, blockIdx.x);
    // copies that may still be in flight must land before the shared memory is reused
    const uint64_t t0 = zb_globaltimer();
    while (zb_globaltimer() - t0 < 200000ull) {
    }
  }
}

// Joins the pairs that several CTAs have a part of.  CTA c looks at the pair at the beginning of part c + 1; the first one to meet a pair there
// joins it, a row of queries in each warp, or in each of two where rows are eight.
template <int HD, int NB>
__global__ void __launch_bounds__(512) zb_kv8_join_kernel(const Kv8DecodeParams p) {
  constexpr int kRows = 8 * NB, kGroups = 16 / kRows, kCols = HD / 32;
  __shared__ float weight[kRows][kMaxCtas];
  __shared__ float sums[kRows];
  __shared__ float parts[kGroups][kRows][HD];
  zb_pdl_launch();
  zb_pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = warp % kRows, part = warp / kRows;
  const int pairs = p.hkv * p.blocks;
  const auto count = [&](int s) { return kv8_span(p, s).tiles * pairs; };
  const int total = kv8_total(p.batch, count);
  const Kv8Parts list(total, p.ctas);
  const int c = static_cast<int>(blockIdx.x), at = list.begin(c + 1), start = list.begin(c);
  if (at >= total || at == start) return;
  int seq, before;
  kv8_locate(p.batch, at, count, seq, before);
  const int tiles = kv8_span(p, seq).tiles, pair = (at - before) / tiles, pair0 = before + pair * tiles;
  if (at == pair0 || start > pair0) return;           // nothing is cut here, or the pair has been met before
  const int n = list.of(pair0 + tiles - 1) - c + 1;   // parts c .. c + n - 1, none of them empty
  const int kvh = pair / p.blocks, row0 = (pair - kvh * p.blocks) * kRows, rows = min(kRows, p.group - row0);
  // the pair is the last segment of part c, unless that begins with it, and the first one of the others
  const int slot0 = 2 * c + (start >= pair0 ? 0 : 1);
  const auto slot_of = [&](int i) { return i == 0 ? slot0 : 2 * (c + i); };
  if (part == 0 && row < rows) {
    float top = kNoScore, sum = 0.f;
    for (int i = lane; i < n; i += 32) {
      const float2 ml = p.part_ml[static_cast<size_t>(slot_of(i)) * kRows + row];
      weight[row][i] = ml.x;
      const float up = fmaxf(top, ml.x);
      sum = sum * zb_ex2(top - up) + ml.y * zb_ex2(ml.x - up);
      top = up;
    }
    const float all = zb_warp_max(top);
    sum = zb_warp_sum(sum * zb_ex2(top - all));
    for (int i = lane; i < n; i += 32) weight[row][i] = zb_ex2(weight[row][i] - all);
    if (lane == 0) sums[row] = sum;
  }
  __syncthreads();
  float acc[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) acc[j] = 0.f;
  if (row < rows) {
#pragma unroll 4
    for (int i = part; i < n; i += kGroups) {
      const float f = weight[row][i];
      const float* src = p.part_o + (static_cast<size_t>(slot_of(i)) * kRows + row) * HD;
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[j] += f * src[lane + 32 * j];
    }
  }
#pragma unroll
  for (int j = 0; j < kCols; ++j) parts[part][row][lane + 32 * j] = acc[j];
  __syncthreads();
  for (int i = threadIdx.x; i < rows * HD; i += 512) {
    const int r = i / HD, col = i - r * HD;
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) x += parts[k][r][col];
    p.out[(static_cast<size_t>(seq) * p.hkv * p.group + kvh * p.group + row0 + r) * HD + col] = __float2bfloat16(sums[r] == 0.f ? 0.f : x / sums[r]);
  }
}

template <int HD, int NB, bool INT8>
int launch_decode(const Kv8DecodeParams& p, const void* k_codes, const void* v_codes, cudaStream_t stream) {
  using Z = Kv8Sizes<HD, NB>;
  static bool configured[16] = {};
  if (const int rc = zb_config_smem_once(zb_kv8_decode_kernel<HD, NB, INT8>, Z::kSmem, configured)) return rc;
  const long long rows = static_cast<long long>(p.num_pages) * p.hkv * p.page_size;
  const int box_rows = HD == 64 ? p.unit / 2 : p.unit;
  CUtensorMap tk, tv;
  const long long map_rows = HD == 64 ? rows / 2 : rows, map_bytes = HD == 64 ? 128 : HD;
  if (const int rc = zb_make_tmap_u8_2d_ex(&tk, k_codes, map_rows, map_bytes, 128, box_rows, 1)) return rc;
  if (const int rc = zb_make_tmap_u8_2d_ex(&tv, v_codes, map_rows, map_bytes, 128, box_rows, 1)) return rc;
  cudaError_t e = zb_launch(zb_kv8_decode_kernel<HD, NB, INT8>, dim3(p.ctas), dim3(160), Z::kSmem, stream, tk, tv, p);
  zb_count_launch(1);
  if (e == cudaSuccess && p.ctas > 1) {
    e = zb_launch(zb_kv8_join_kernel<HD, NB>, dim3(p.ctas - 1), dim3(512), 0, stream, p);
    zb_count_launch(1);
  }
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

// Query heads of a pair: 16 where the group has more than eight (a head of 256 has registers for eight).
int rows_of(int hd, int group) { return group > 8 && hd <= 128 ? 16 : 8; }
int per_sm_of(int hd, int rows) {
  if (hd == 64) return rows == 8 ? Kv8Sizes<64, 1>::kPerSm : Kv8Sizes<64, 2>::kPerSm;
  if (hd == 128) return rows == 8 ? Kv8Sizes<128, 1>::kPerSm : Kv8Sizes<128, 2>::kPerSm;
  return Kv8Sizes<256, 1>::kPerSm;
}

}  // namespace

extern "C" {

// CTAs of a call, and (in *floats) the fp32 numbers of its workspace.  max_len: keys of the longest sequence, or a bound of them: it bounds the
// CTAs that have something to do, any number gives right results.
int zb_kv8_decode_plan(int batch, int hq, int hkv, int hd, int max_len, long long* floats) {
  *floats = 0;
  if (batch <= 0) return 0;
  if (hkv <= 0 || hq <= 0 || hq % hkv != 0 || (hd != 64 && hd != 128 && hd != 256)) return -30;
  ZbDeviceState* st = zb_device_state();
  if (!st) return -20;
  const int rows = rows_of(hd, hq / hkv), blocks = (hq / hkv + rows - 1) / rows;
  const long long tiles = static_cast<long long>(batch) * hkv * blocks * std::max(1, (max_len + kTile - 1) / kTile);
  if (tiles > 0x3fffffffll) return -34;
  const int ctas = static_cast<int>(std::min<long long>(tiles, std::min(kMaxCtas, st->num_sms * per_sm_of(hd, rows))));
  *floats = 2ll * ctas * rows * (hd + 2);
  return ctas;
}

// The arguments of a call, as the caller packs them (ops/kv8.py).
struct ZbKv8Decode {
  const void* q;                                   // [batch, hq, hd], rows on 8 bytes
  const void *k_codes, *k_exps, *v_codes, *v_exps;  // contiguous, on 16 bytes
  void* out;                                       // [batch, hq, hd], contiguous
  const int32_t* block_table;
  const int32_t* seq_lens;
  float* work;                                     // the numbers that the plan of `ctas` CTAs asked for
  void* stream;
  long long q_stride;
  int batch, hq, hkv, hd, page_size, max_pages, num_pages, window, int8, ctas;
  float scale;
};

int zb_kv8_decode(const ZbKv8Decode* c) {
  const int hq = c->hq, hkv = c->hkv, hd = c->hd, page_size = c->page_size;
  if (c->batch <= 0) return 0;
  if (hkv <= 0 || hq <= 0 || hq % hkv != 0 || (hd != 64 && hd != 128 && hd != 256)) return -30;
  if (page_size <= 0 || page_size % 16 != 0 || c->num_pages <= 0 || static_cast<long long>(c->num_pages) * hkv * page_size > 0x7fffffffll ||
      static_cast<long long>(c->max_pages) * page_size > 0x7fffff00ll)
    return -31;
  if (c->ctas < 1 || c->ctas > kMaxCtas) return -33;
  ZbDeviceState* st = zb_device_state();
  if (!st) return -20;
  const int rows = rows_of(hd, hq / hkv);
  Kv8DecodeParams p = {};
  p.q = reinterpret_cast<const __nv_bfloat16*>(c->q);
  p.k_exps = reinterpret_cast<const uint8_t*>(c->k_exps);
  p.v_exps = reinterpret_cast<const uint8_t*>(c->v_exps);
  p.out = reinterpret_cast<__nv_bfloat16*>(c->out);
  p.block_table = c->block_table;
  p.seq_lens = c->seq_lens;
  p.part_o = c->work;
  p.part_ml = reinterpret_cast<float2*>(c->work + 2ll * c->ctas * rows * hd);
  p.q_stride = c->q_stride;
  p.batch = c->batch;
  p.hkv = hkv;
  p.group = hq / hkv;
  p.blocks = (p.group + rows - 1) / rows;
  p.page_size = page_size;
  p.max_pages = c->max_pages;
  p.num_pages = c->num_pages;
  p.window = c->window;
  p.unit = 16;
  while (p.unit < kTile && page_size % (2 * p.unit) == 0) p.unit *= 2;
  p.ctas = c->ctas;
  p.scale_log2 = c->scale * 1.4426950408889634f;
  p.status = st->status;
  if (static_cast<long long>(c->batch) * hkv * p.blocks * std::max<long long>(1, (static_cast<long long>(c->max_pages) * page_size + kTile - 1) / kTile) > 0x3fffffffll)
    return -34;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(c->stream);
  const void *k = c->k_codes, *v = c->v_codes;
  const bool int8 = c->int8 != 0;
  if (hd == 64) {
    if (rows == 8) return int8 ? launch_decode<64, 1, true>(p, k, v, s) : launch_decode<64, 1, false>(p, k, v, s);
    return int8 ? launch_decode<64, 2, true>(p, k, v, s) : launch_decode<64, 2, false>(p, k, v, s);
  }
  if (hd == 128) {
    if (rows == 8) return int8 ? launch_decode<128, 1, true>(p, k, v, s) : launch_decode<128, 1, false>(p, k, v, s);
    return int8 ? launch_decode<128, 2, true>(p, k, v, s) : launch_decode<128, 2, false>(p, k, v, s);
  }
  return int8 ? launch_decode<256, 1, true>(p, k, v, s) : launch_decode<256, 1, false>(p, k, v, s);
}

}  // extern "C"
