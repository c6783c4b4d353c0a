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
//   [2^13, 2^14), exactly, and that power is taken out of its scores; s_vj is taken relative to the largest one so far, which rescales the
//   accumulators like the maximum of the scores does.  What f16 drops lies 2^-25 below the largest weight.
// * All tiles of 64 keys of all (sequence, key head) pairs are one list, cut into equal parts, one for each CTA: whatever the mix of lengths,
//   all SMs stream alike.  A CTA whose part ends inside a pair leaves its sums in the workspace, and a second kernel joins each such
//   pair.  Lengths are read on the device, so a captured launch serves any of them; nothing outlives the two launches.
// * Four warps take 16 keys of a tile each; a fifth one feeds the ring of tiles, page numbers fetched 32 at a time.
#include <cuda.h>

#include <algorithm>

#include "host_api.h"
#include "kv8.cuh"

int zb_make_tmap_u8_2d_ex(CUtensorMap* out, const void* base, long long rows, long long row_bytes, int box_bytes, int box_rows, int swizzle128);

namespace {

constexpr uint32_t kKernelKv8Decode = 41;
constexpr int kTile = 64;                       // keys
constexpr int kMaxCtas = 384;                   // of the partition: what the joining kernel keeps weights for

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
// First position of CTA c's part of `total`.
ZB_DEVICE int kv8_part(int total, int c, int ctas) { return static_cast<int>(static_cast<long long>(total) * c / ctas); }

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
  w.at = kv8_part(total, blockIdx.x, p.ctas);
  w.last = kv8_part(total, blockIdx.x + 1, p.ctas);
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
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
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
          if (dead || lane != 0) continue;
          const long long row = (static_cast<long long>(page) * p.hkv + kvh) * p.page_size + (key0 + c * p.unit) % p.page_size;
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
      float m[NB][2], l[NB][2];
#pragma unroll
      for (int b = 0; b < NB; ++b) m[b][0] = m[b][1] = -INFINITY, l[b][0] = l[b][1] = 0.f;
      uint32_t power = 1u;                            // exponent byte of the largest scale of a value so far

      for (int t = w.begin; t < w.end; ++t) {
        if (!dead) dead = !zb_mbar_wait(&full_bar[stage], phase, abort_flag);
        dead = __any_sync(0xffffffffu, dead);
        const int key0 = (w.span.tile0 + t) * kTile + warp * 16;
        if (!dead && key0 < w.span.len && key0 + 16 > w.span.first) {
          const uint8_t* ks = smem + stage * Z::kStageBytes;
          const uint8_t* vs = ks + Z::kTileBytes;
          const uint8_t* ex = exps + stage * 2 * kTile + warp * 16;
          const bool whole = key0 >= w.span.first && key0 + 16 <= w.span.len;
          // S^T: keys g and g + 8 of the 16
          float s[NB][4];
#pragma unroll
          for (int b = 0; b < NB; ++b) s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
          const int r0 = warp * 16 + g, r1 = r0 + 8;
#pragma unroll
          for (int c = 0; c < kSteps / 4; ++c) {
            uint4 x, y;
            if constexpr (HD == 64) {
              x = *reinterpret_cast<const uint4*>(ks + (r0 >> 1) * 128 + (((((r0 & 1) << 2) + t4) ^ ((r0 >> 1) & 7)) << 4));
              y = *reinterpret_cast<const uint4*>(ks + (r1 >> 1) * 128 + (((((r1 & 1) << 2) + t4) ^ ((r1 >> 1) & 7)) << 4));
            } else {
              const int at = (c >> 1) * kTile * 128 + (((2 * t4 + (c & 1)) ^ (r0 & 7)) << 4);
              x = *reinterpret_cast<const uint4*>(ks + at + r0 * 128);
              y = *reinterpret_cast<const uint4*>(ks + at + r1 * 128);
            }
            const uint32_t wx[4] = {x.x, x.y, x.z, x.w}, wy[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a0, a1, a2, a3;
              kv8_to_half<INT8>(wx[i], a0, a2);
              kv8_to_half<INT8>(wy[i], a1, a3);
#pragma unroll
              for (int b = 0; b < NB; ++b) mma_f16(s[b], a0, a1, a2, a3, qf[b][c * 4 + i][0], qf[b][c * 4 + i][1]);
            }
          }
          const bool see0 = whole || (key0 + g >= w.span.first && key0 + g < w.span.len);
          const bool see1 = whole || (key0 + g + 8 >= w.span.first && key0 + g + 8 < w.span.len);
          const float ks0 = kv8_scale(ex[g]), ks1 = kv8_scale(ex[g + 8]);
          const uint32_t ve0 = see0 ? ex[kTile + g] : 0u, ve1 = see1 ? ex[kTile + g + 8] : 0u;
          // values' scales relative to the largest one so far; 255 (a row that is NaN) stays an infinity and its codes of zero make a NaN of it
          const uint32_t now = max(power, __reduce_max_sync(0xffffffffu, min(max(ve0, ve1), 253u)));
          const float shrink = power == now ? 1.f : (now - power > 126u ? 0.f : __uint_as_float((127u - (now - power)) << 23));
          power = now;
          const float unit = __uint_as_float((254u - now) << 23), vs0 = kv8_scale(ve0) * unit, vs1 = kv8_scale(ve1) * unit;
          float corr[NB][2];
          bool moved = shrink != 1.f;
          uint32_t pb[NB][2];
#pragma unroll
          for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              s[b][j] = see0 ? s[b][j] * (ks0 * factor[b][j]) : -INFINITY;
              s[b][j + 2] = see1 ? s[b][j + 2] * (ks1 * factor[b][j]) : -INFINITY;
              float mx = fmaxf(s[b][j], s[b][j + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float mnew = fmaxf(m[b][j], mx), use = mnew == -INFINITY ? 0.f : mnew;
              const float c = exp2f(m[b][j] - use);
              m[b][j] = mnew;
              s[b][j] = exp2f(s[b][j] - use);
              s[b][j + 2] = exp2f(s[b][j + 2] - use);
              l[b][j] = l[b][j] * c + (s[b][j] + s[b][j + 2]);
              corr[b][j] = c * shrink;
              moved = moved || c != 1.f;
            }
            pb[b][0] = transpose8(pack_half2(see0 ? s[b][0] * vs0 : 0.f, see0 ? s[b][1] * vs0 : 0.f));
            pb[b][1] = transpose8(pack_half2(see1 ? s[b][2] * vs1 : 0.f, see1 ? s[b][3] * vs1 : 0.f));
          }
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[b][i][j] *= corr[b][j & 1];
          }
          // O^T: keys 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9 of the 16; columns: piece g of each half row (HD 64: half a piece)
#pragma unroll
          for (int sub = 0; sub < kSubs; ++sub) {
            uint32_t v[4][HD == 64 ? 2 : 4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int kk = 2 * t4 + (k & 1) + (k >> 1) * 8, r = warp * 16 + kk;
              if constexpr (HD == 64) {
                const uint2 x = *reinterpret_cast<const uint2*>(vs + (r >> 1) * 128 + (((((r & 1) << 2) + (g >> 1)) ^ ((r >> 1) & 7)) << 4) + (g & 1) * 8);
                v[k][0] = x.x, v[k][1] = x.y;
              } else {
                const uint4 x = *reinterpret_cast<const uint4*>(vs + sub * kTile * 128 + r * 128 + ((g ^ (r & 7)) << 4));
                v[k][0] = x.x, v[k][1] = x.y, v[k][2] = x.z, v[k][3] = x.w;
              }
              // codes of rows that nobody sees may be anything, e4m3's NaN, too
              if (!whole && (key0 + kk < w.span.first || key0 + kk >= w.span.len)) {
#pragma unroll
                for (int i = 0; i < (HD == 64 ? 2 : 4); ++i) v[k][i] = 0u;
              }
            }
#pragma unroll
            for (int i = 0; i < (HD == 64 ? 2 : 4); ++i) {
              // pairs of keys of each of the word's four columns
              uint32_t a[4], c[4];
              kv8_to_half<INT8>(__byte_perm(v[0][i], v[1][i], 0x5140), a[0], a[1]);
              kv8_to_half<INT8>(__byte_perm(v[2][i], v[3][i], 0x5140), a[2], a[3]);
              kv8_to_half<INT8>(__byte_perm(v[0][i], v[1][i], 0x7362), c[0], c[1]);
              kv8_to_half<INT8>(__byte_perm(v[2][i], v[3][i], 0x7362), c[2], c[3]);
#pragma unroll
              for (int b = 0; b < NB; ++b) {
                mma_f16(o[b][sub * 8 + 2 * i], a[0], a[1], a[2], a[3], pb[b][0], pb[b][1]);
                mma_f16(o[b][sub * 8 + 2 * i + 1], c[0], c[1], c[2], c[3], pb[b][0], pb[b][1]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) zb_mbar_arrive(&empty_bar[stage]);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }

      // the four warps' sums of this segment
      const float power_of = __uint_as_float(power << 23);
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
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, stats[(k * kRows + r) * 3]);
        const float use = top == -INFINITY ? 0.f : top;
        float ax = 0.f, ay = 0.f, sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float* st = stats + (k * kRows + r) * 3;
          const float f = exp2f(st[0] - use), fo = f * st[2];
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
// joins it, a row of queries for eight or 16 of its 32 warps at a time.
template <int HD, int NB>
__global__ void __launch_bounds__(1024) zb_kv8_join_kernel(const Kv8DecodeParams p) {
  constexpr int kRows = 8 * NB, kGroups = 32 / kRows, kCols = HD / 32;
  __shared__ float weight[kRows][kMaxCtas];
  __shared__ float sums[kRows];
  __shared__ float parts[kGroups][kRows][HD];
  zb_pdl_launch();
  zb_pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = warp % kRows, part = warp / kRows;
  const int pairs = p.hkv * p.blocks;
  const auto count = [&](int s) { return kv8_span(p, s).tiles * pairs; };
  const int total = kv8_total(p.batch, count);
  const int c = static_cast<int>(blockIdx.x), at = kv8_part(total, c + 1, p.ctas), start = kv8_part(total, c, p.ctas);
  if (at >= total || at == start) return;
  int seq, before;
  kv8_locate(p.batch, at, count, seq, before);
  const int tiles = kv8_span(p, seq).tiles, pair = (at - before) / tiles, pair0 = before + pair * tiles, pair1 = pair0 + tiles;
  if (at == pair0 || start > pair0) return;           // nothing is cut here, or the pair has been met before
  const int end = static_cast<int>((static_cast<long long>(pair1) * p.ctas - 1) / total);      // the last part that begins in front of pair1
  const int n = end - c + 1;
  const int kvh = pair / p.blocks, row0 = (pair - kvh * p.blocks) * kRows, rows = min(kRows, p.group - row0);
  const auto slot_of = [&](int i) {                   // -1: an empty part
    const int x = kv8_part(total, c + i, p.ctas);
    return x == kv8_part(total, c + i + 1, p.ctas) ? -1 : 2 * (c + i) + (x >= pair0 ? 0 : 1);
  };
  if (part == 0 && row < rows) {
    float top = -INFINITY;
    for (int i = lane; i < n; i += 32) {
      const int s = slot_of(i);
      const float m = s < 0 ? -INFINITY : p.part_ml[static_cast<size_t>(s) * kRows + row].x;
      weight[row][i] = m;
      top = fmaxf(top, m);
    }
    top = zb_warp_max(top);
    const float use = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int i = lane; i < n; i += 32) {
      const int s = slot_of(i);
      const float f = exp2f(weight[row][i] - use);
      weight[row][i] = f;
      if (s >= 0) sum += f * p.part_ml[static_cast<size_t>(s) * kRows + row].y;
    }
    sum = zb_warp_sum(sum);
    if (lane == 0) sums[row] = sum;
  }
  __syncthreads();
  float acc[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) acc[j] = 0.f;
  if (row < rows) {
#pragma unroll 4
    for (int i = part; i < n; i += kGroups) {
      const int s = slot_of(i);
      if (s < 0) continue;
      const float f = weight[row][i];
      const float* src = p.part_o + (static_cast<size_t>(s) * kRows + row) * HD;
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[j] += f * src[lane + 32 * j];
    }
  }
#pragma unroll
  for (int j = 0; j < kCols; ++j) parts[part][row][lane + 32 * j] = acc[j];
  __syncthreads();
  for (int i = threadIdx.x; i < rows * HD; i += 1024) {
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
    e = zb_launch(zb_kv8_join_kernel<HD, NB>, dim3(p.ctas - 1), dim3(1024), 0, stream, p);
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

// q [batch, hq, hd] with q_stride elements between rows, which start on 8 bytes; out [batch, hq, hd]; codes and exponents start on 16 bytes;
// `work`: the numbers that the plan of `ctas` CTAs asked for.
int zb_kv8_decode(const void* q, const void* k_codes, const void* k_exps, const void* v_codes, const void* v_exps, void* out,
                  const int32_t* block_table, const int32_t* seq_lens, int batch, int hq, int hkv, int hd, int page_size, int max_pages,
                  int num_pages, long long q_stride, float scale, int window, int int8, float* work, int ctas, void* stream) {
  if (batch <= 0) return 0;
  if (hkv <= 0 || hq <= 0 || hq % hkv != 0 || (hd != 64 && hd != 128 && hd != 256)) return -30;
  if (page_size <= 0 || page_size % 16 != 0 || num_pages <= 0 || static_cast<long long>(num_pages) * hkv * page_size > 0x7fffffffll ||
      static_cast<long long>(max_pages) * page_size > 0x7fffff00ll)
    return -31;
  if (ctas < 1 || ctas > kMaxCtas) return -33;
  ZbDeviceState* st = zb_device_state();
  if (!st) return -20;
  const int rows = rows_of(hd, hq / hkv);
  Kv8DecodeParams p = {};
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.k_exps = reinterpret_cast<const uint8_t*>(k_exps);
  p.v_exps = reinterpret_cast<const uint8_t*>(v_exps);
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.part_o = work;
  p.part_ml = reinterpret_cast<float2*>(work + 2ll * ctas * rows * hd);
  p.q_stride = q_stride;
  p.batch = batch;
  p.hkv = hkv;
  p.group = hq / hkv;
  p.blocks = (p.group + rows - 1) / rows;
  p.page_size = page_size;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.window = window;
  p.unit = 16;
  while (p.unit < kTile && page_size % (2 * p.unit) == 0) p.unit *= 2;
  p.ctas = ctas;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = st->status;
  if (static_cast<long long>(batch) * hkv * p.blocks * std::max<long long>(1, (static_cast<long long>(max_pages) * page_size + kTile - 1) / kTile) > 0x3fffffffll)
    return -34;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (hd == 64) {
    if (rows == 8) return int8 ? launch_decode<64, 1, true>(p, k_codes, v_codes, s) : launch_decode<64, 1, false>(p, k_codes, v_codes, s);
    return int8 ? launch_decode<64, 2, true>(p, k_codes, v_codes, s) : launch_decode<64, 2, false>(p, k_codes, v_codes, s);
  }
  if (hd == 128) {
    if (rows == 8) return int8 ? launch_decode<128, 1, true>(p, k_codes, v_codes, s) : launch_decode<128, 1, false>(p, k_codes, v_codes, s);
    return int8 ? launch_decode<128, 2, true>(p, k_codes, v_codes, s) : launch_decode<128, 2, false>(p, k_codes, v_codes, s);
  }
  return int8 ? launch_decode<256, 1, true>(p, k_codes, v_codes, s) : launch_decode<256, 1, false>(p, k_codes, v_codes, s);
}

}  // extern "C"
