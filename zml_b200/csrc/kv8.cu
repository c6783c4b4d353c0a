// Writer and reader of the paged key / value cache in 8 bits (format: kv8.cuh).
//
//   zb_kv8_write   one pass over the fused projection [T, (Hq + 2 Hkv) * HD]: optional RMSNorm of every query and key head, rotation by
//                  the token's position, queries to bf16, keys and values to codes and exponents at their slots
//   zb_kv8_read    whole sequences out of their pages into dense bf16 pages [pages, page_size, Hkv, HD], and the block table of those
//
// Between the bf16 projection and the one rounding at the end (bf16 queries, codes) everything is fp32: a rounding to bf16 in between would put
// three codes of a hundred into the neighbouring step.  Angles p * f are formed and reduced in fp64 (one per pair of columns and token, used
// by all heads), so that far positions keep the digits that fp32 products lose (1e5 radians: 0.004).
#include <algorithm>

#include "host_api.h"
#include "kv8.cuh"

namespace {

constexpr uint32_t kKernelKv8Write = 39, kKernelKv8Read = 40;

struct Kv8WriteParams {
  const __nv_bfloat16* qkv;
  __nv_bfloat16* q_out;
  uint8_t* k_codes;
  uint8_t* v_codes;
  uint8_t* k_exps;
  uint8_t* v_exps;
  const int32_t* positions;
  const int32_t* slot_mapping;
  const float* inv_freq;
  const __nv_bfloat16* q_norm_w;
  const __nv_bfloat16* k_norm_w;
  long long qkv_stride, num_slots;
  int tokens, hq, hkv, hd, rot_dim, layout, page_size;
  float attn_factor, norm_eps;
  int norm_unit_offset;
  int share;                   // pieces of a token that one CTA takes
  ZbStatus* status;
};

// cos and sin of position * frequency, each rounded once to fp32.  The angle is formed in fp64 and taken back to [-pi/4, pi/4] by a multiple of pi/2 in
// two parts; there the Taylor series up to r^13 and r^12 leave 2^-40.  About 20 fp64 operations, which cost less than fp32's own functions do.
ZB_DEVICE void kv8_angle(int pos, float freq, float factor, float& sn, float& cs) {
  const double a = static_cast<double>(pos) * static_cast<double>(freq);
  const double n = rint(a * 0.6366197723675814);
  const double r = fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, a)), x = r * r;
  const double s = r * fma(x, fma(x, fma(x, fma(x, fma(x, fma(x, 1.6059043836821613e-10, -2.505210838544172e-08), 2.7557319223985893e-06), -1.984126984126984e-04),
                                         8.333333333333333e-03), -1.6666666666666666e-01), 1.0);
  const double c = fma(x, fma(x, fma(x, fma(x, fma(x, fma(x, 2.08767569878681e-09, -2.755731922398589e-07), 2.48015873015873e-05), -1.388888888888889e-03),
                                     4.1666666666666664e-02), -0.5), 1.0);
  const int q = static_cast<int>(static_cast<long long>(n) & 3);
  const float fs = static_cast<float>((q & 1) ? c : s), fc = static_cast<float>((q & 1) ? s : c);
  sn = ((q & 2) ? -fs : fs) * factor;
  cs = ((q == 1 || q == 2) ? -fc : fc) * factor;
}

// Slot of token `tok`: -1 for a token that writes nothing.  One behind the cache is reported.
ZB_DEVICE long long kv8_slot(const Kv8WriteParams& p, int tok) {
  const long long slot = p.slot_mapping[tok];
  if (slot >= p.num_slots) {
    zb_record_error(p.status, ZB_ERR_BOUNDS, kKernelKv8Write, 1u, static_cast<uint32_t>(slot));
    return -1;
  }
  return slot < 0 ? -1 : slot;
}

// Row of head kvh at a slot, in units of rows.
ZB_DEVICE size_t kv8_row_at(const Kv8WriteParams& p, long long slot, int kvh) {
  const int page = static_cast<int>(slot) / p.page_size, off = static_cast<int>(slot) % p.page_size;
  return (static_cast<size_t>(page) * p.hkv + kvh) * p.page_size + off;
}

ZB_DEVICE void kv8_unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = zb_unpack_bf16x2(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

// Halves (LAYOUT 0, rot_dim a multiple of 16) or neighbours (LAYOUT 1) rotate into each other; rows start on 16 bytes.  A thread has two pieces of
// eight columns of one head, the same of every token: the two that rotate into each other, or two neighbours.  The HD / 16 threads of a head lie in
// one warp and add up its squares and its largest magnitude.  A CTA takes one token after the other (its threads a part of the pieces where those are more
// than 512): the next projection is on its way while it works on this one, and its threads form the angles and the cache rows of kAhead tokens at
// once, one or two each, so that they meet once in as many tokens.
// Numbers go in packed pairs, which halves the arithmetic: the kernel is bound by its instructions as much as by memory.  8192 tokens of 32 / 4 normed heads of
// 128 take 30.4 us, 5.2 TB/s (80 % of a copy's rate); 34.1 where every thread finds its row, 38 with the loop over kAhead tokens unrolled.
constexpr int kAhead = 4;
ZB_DEVICE ZbF2 kv8_pair(uint32_t bf16x2) {
  const float2 v = zb_unpack_bf16x2(bf16x2);
  return zb_pack2(v.x, v.y);
}
ZB_DEVICE uint32_t kv8_bf16x2(ZbF2 v) {
  float x, y;
  zb_unpack2(v, x, y);
  return zb_pack_bf16x2(x, y);
}
ZB_DEVICE uint32_t kv8_abs_max(uint32_t most, ZbF2 v) {
  float x, y;
  zb_unpack2(v, x, y);
  return max(most, max(kv8_abs_bits(x), kv8_abs_bits(y)));
}
template <bool INT8>
ZB_DEVICE uint32_t kv8_codes4(ZbF2 inv, ZbF2 a, ZbF2 b, bool finite) {
  float x0, x1, x2, x3;
  zb_unpack2(zb_mul2(a, inv), x0, x1);
  zb_unpack2(zb_mul2(b, inv), x2, x3);
  return finite ? kv8_pack4<INT8>(1.f, x0, x1, x2, x3) : 0u;
}

template <int HD, int LAYOUT, bool INT8>
__global__ void __launch_bounds__(512, 2) zb_kv8_write_kernel(const Kv8WriteParams p) {
  constexpr int kLanes = HD / 16, kHalf = HD / 2;
  // cosines and sines; angle i lies where a thread's eight are two pieces of 16 bytes, neighbouring threads' beside each other
  __shared__ __align__(16) float cs[2][kAhead][kHalf], sn[2][kAhead][kHalf];
  __shared__ __align__(16) float weights[2][HD];       // of queries' and keys' norms, laid out alike
  __shared__ long long rows[2][kAhead];
  zb_pdl_launch();
  zb_pdl_wait();
  const int half = p.rot_dim >> 1;
  const int units = (p.hq + 2 * p.hkv) * kLanes, u = min(static_cast<int>(blockIdx.y) * p.share + static_cast<int>(threadIdx.x), units - 1);
  const bool in = static_cast<int>(threadIdx.x) < p.share && static_cast<int>(blockIdx.y) * p.share + static_cast<int>(threadIdx.x) < units;
  const int h = u / kLanes, j = u - h * kLanes;
  const bool is_q = h < p.hq, turned = h < p.hq + p.hkv, turns = turned && (LAYOUT == 1 || j < half / 8);
  const int a0 = LAYOUT == 1 || !turned ? 2 * j : (turns ? j : half / 4 + 2 * (j - half / 8));
  const int a1 = LAYOUT == 0 && turns ? j + half / 8 : a0 + 1;
  const bool any_kv = __any_sync(0xffffffffu, !is_q);
  const uint4* src = reinterpret_cast<const uint4*>(p.qkv + static_cast<size_t>(h) * HD);
  const bool normed = turned && (is_q ? p.q_norm_w : p.k_norm_w) != nullptr, any_normed = __any_sync(0xffffffffu, normed);
  const int kvh = turned ? h - p.hq : h - p.hq - p.hkv;
  uint8_t* const codes = turned ? p.k_codes : p.v_codes;
  uint8_t* const exps = turned ? p.k_exps : p.v_exps;

  // angles of the next kAhead tokens of this CTA, and the rows of head 0 that they write (negative: none)
  const auto ahead = [&](long long from, int buf) {
    for (int i = threadIdx.x; i < kAhead * half; i += blockDim.x) {
      const int k = i / half, n = i - k * half;
      const long long tok = from + static_cast<long long>(k) * gridDim.x;
      if (tok >= p.tokens) break;
      const int at = ((n >> 2) & 1) * (kHalf / 2) + (n >> 3) * 4 + (n & 3);
      kv8_angle(p.positions[tok], p.inv_freq[n], p.attn_factor, sn[buf][k][at], cs[buf][k][at]);
    }
    const long long tok = from + static_cast<long long>(blockDim.x - 1 - threadIdx.x) * gridDim.x;
    if (blockDim.x - 1 - threadIdx.x < kAhead && tok < p.tokens) {
      const long long slot = kv8_slot(p, static_cast<int>(tok));
      rows[buf][blockDim.x - 1 - threadIdx.x] = slot < 0 ? -1ll : static_cast<long long>(kv8_row_at(p, slot, 0));
    }
  };
  int buf = 0;
  long long tok = blockIdx.x;
  uint4 x0 = src[static_cast<size_t>(tok) * p.qkv_stride / 8 + a0], x1 = src[static_cast<size_t>(tok) * p.qkv_stride / 8 + a1];
  for (int i = threadIdx.x; i < 2 * HD; i += blockDim.x) {
    const __nv_bfloat16* w = i < HD ? p.q_norm_w : p.k_norm_w;
    const int n = i % HD;
    if (w != nullptr) weights[i / HD][((n >> 2) & 1) * kHalf + (n >> 3) * 4 + (n & 3)] = __bfloat162float(w[n]) + (p.norm_unit_offset ? 1.f : 0.f);
  }
  ahead(tok, 0);
  __syncthreads();
  const auto step = [&](int k) {                       // false: that was the last token
    const long long tok1 = tok + gridDim.x;
    const bool more = tok1 < p.tokens;
    ZbF2 f0[4] = {kv8_pair(x0.x), kv8_pair(x0.y), kv8_pair(x0.z), kv8_pair(x0.w)}, f1[4] = {kv8_pair(x1.x), kv8_pair(x1.y), kv8_pair(x1.z), kv8_pair(x1.w)};
    if (more) {
      const uint4* from = src + static_cast<size_t>(tok1) * p.qkv_stride / 8;
      x0 = from[a0], x1 = from[a1];
    }
    if (k == 0 && tok + static_cast<long long>(kAhead) * gridDim.x < p.tokens) ahead(tok + static_cast<long long>(kAhead) * gridDim.x, buf ^ 1);
    if (any_normed) {
      ZbF2 sum = zb_mul2(f0[0], f0[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) sum = zb_fma2(f0[i], f0[i], sum);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = zb_fma2(f1[i], f1[i], sum);
      float ss = zb_sum2(sum);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (normed) {
        const float inv = rsqrtf(ss / static_cast<float>(HD) + p.norm_eps);
        const ZbF2 by = zb_pack2(inv, inv);
        const ulonglong2* w = reinterpret_cast<const ulonglong2*>(weights[is_q ? 0 : 1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const ulonglong2 g0 = w[i * (HD / 8) + a0], g1 = w[i * (HD / 8) + a1];
          f0[2 * i] = zb_mul2(zb_mul2(f0[2 * i], by), g0.x), f0[2 * i + 1] = zb_mul2(zb_mul2(f0[2 * i + 1], by), g0.y);
          f1[2 * i] = zb_mul2(zb_mul2(f1[2 * i], by), g1.x), f1[2 * i + 1] = zb_mul2(zb_mul2(f1[2 * i + 1], by), g1.y);
        }
      }
    }
    if (turns) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&cs[buf][k][q * (kHalf / 2) + 4 * j]), s = *reinterpret_cast<const ulonglong2*>(&sn[buf][k][q * (kHalf / 2) + 4 * j]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const ZbF2 ci = i ? c.y : c.x, si = i ? s.y : s.x;
          if (LAYOUT == 0) {
            ZbF2& x = f0[2 * q + i];
            ZbF2& y = f1[2 * q + i];
            const ZbF2 a = x, b = y;
            x = zb_fma2(a, ci, zb_mul2(b, si ^ 0x8000000080000000ull));
            y = zb_fma2(b, ci, zb_mul2(a, si));
          } else {
            float c0, c1, s0, s1, a, b;
            zb_unpack2(ci, c0, c1);
            zb_unpack2(si, s0, s1);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              ZbF2& v = q == 0 ? f0[2 * i + e] : f1[2 * i + e];
              zb_unpack2(v, a, b);
              const float cc = e ? c1 : c0, ss = e ? s1 : s0;
              if (8 * j + 4 * q + 2 * i + e < half) v = zb_pack2(a * cc - b * ss, b * cc + a * ss);
            }
          }
        }
      }
    }
    if (is_q && in) {
      uint4* dst = reinterpret_cast<uint4*>(p.q_out + (static_cast<size_t>(tok) * p.hq + h) * HD);
      dst[a0] = make_uint4(kv8_bf16x2(f0[0]), kv8_bf16x2(f0[1]), kv8_bf16x2(f0[2]), kv8_bf16x2(f0[3]));
      dst[a1] = make_uint4(kv8_bf16x2(f1[0]), kv8_bf16x2(f1[1]), kv8_bf16x2(f1[2]), kv8_bf16x2(f1[3]));
    }
    if (any_kv) {
      uint32_t amax = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = kv8_abs_max(kv8_abs_max(amax, f0[i]), f1[i]);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const long long row = rows[buf][k];
      if (!is_q && in && row >= 0) {
        const uint32_t byte = kv8_exponent<INT8>(amax);
        const bool finite = byte != 255u;
        const float by = kv8_inverse(byte);
        const ZbF2 inv = zb_pack2(by, by);
        const size_t at = static_cast<size_t>(row) + static_cast<size_t>(kvh) * p.page_size;
        uint2* dst = reinterpret_cast<uint2*>(codes + at * HD);
        uint2 c0 = make_uint2(kv8_codes4<INT8>(inv, f0[0], f0[1], finite), kv8_codes4<INT8>(inv, f0[2], f0[3], finite));
        uint2 c1 = make_uint2(kv8_codes4<INT8>(inv, f1[0], f1[1], finite), kv8_codes4<INT8>(inv, f1[2], f1[3], finite));
        if (byte == kv8_top<INT8>()) {
          c0 = make_uint2(kv8_below_top<INT8>(c0.x), kv8_below_top<INT8>(c0.y));
          c1 = make_uint2(kv8_below_top<INT8>(c1.x), kv8_below_top<INT8>(c1.y));
        }
        dst[a0] = c0;
        dst[a1] = c1;
        if (j == 0) exps[at] = static_cast<uint8_t>(byte);
      }
    }
    tok = tok1;
    return more;
  };
  while (true) {
#pragma unroll 1
    for (int k = 0; k < kAhead; ++k)
      if (!step(k)) return;
    __syncthreads();                                   // the next angles are there, and these have been read
    buf ^= 1;
  }
}

// Any even rot_dim, all layouts, rows at any address: one warp per head, columns lane, lane + 32, ...; the rotation partner comes
// through shared memory.  Layout 2 pairs i with HD / 2 + i for i < rot_dim / 2.
template <bool INT8>
__global__ void __launch_bounds__(256) zb_kv8_write_any_kernel(const Kv8WriteParams p) {
  __shared__ float sn[128], cs[128], rows[8][256];
  zb_pdl_launch();
  zb_pdl_wait();
  const int tok = blockIdx.x, half = p.rot_dim >> 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = p.hd;
  const long long slot = kv8_slot(p, tok);
  for (int i = threadIdx.x; i < half; i += blockDim.x) kv8_angle(p.positions[tok], p.inv_freq[i], p.attn_factor, sn[i], cs[i]);
  __syncthreads();
  float* x = rows[warp];
  for (int h = warp; h < p.hq + 2 * p.hkv; h += 8) {
    const __nv_bfloat16* src = p.qkv + static_cast<size_t>(tok) * p.qkv_stride + static_cast<size_t>(h) * hd;
    const bool is_q = h < p.hq, turned = h < p.hq + p.hkv;
    const __nv_bfloat16* nw = is_q ? p.q_norm_w : p.k_norm_w;
    float ss = 0.f;
    __syncwarp();
    for (int i = lane; i < hd; i += 32) {
      x[i] = __bfloat162float(src[i]);
      ss += x[i] * x[i];
    }
    if (turned && nw != nullptr) {
      const float inv = rsqrtf(zb_warp_sum(ss) / static_cast<float>(hd) + p.norm_eps);
      for (int i = lane; i < hd; i += 32) x[i] = x[i] * inv * (__bfloat162float(nw[i]) + (p.norm_unit_offset ? 1.f : 0.f));
    }
    __syncwarp();
    float f[8];
    uint32_t amax = 0u;
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      const int i = lane + 32 * a;
      f[a] = 0.f;
      if (i >= hd) continue;
      f[a] = x[i];
      if (turned) {
        const int b = p.layout == 1 ? i >> 1 : (p.layout == 0 ? (i < half ? i : i - half) : (i < hd / 2 ? i : i - hd / 2));
        const bool second = p.layout == 1 ? (i & 1) != 0 : (p.layout == 0 ? i >= half : i >= hd / 2);
        if (b < half) {
          const int o = p.layout == 1 ? i ^ 1 : (p.layout == 0 ? (second ? i - half : i + half) : (second ? i - hd / 2 : i + hd / 2));
          f[a] = second ? f[a] * cs[b] + x[o] * sn[b] : f[a] * cs[b] - x[o] * sn[b];
        }
      }
      amax = max(amax, kv8_abs_bits(f[a]));
    }
    if (is_q) {
      for (int a = 0; a < hd / 32; ++a) p.q_out[(static_cast<size_t>(tok) * p.hq + h) * hd + lane + 32 * a] = __float2bfloat16(f[a]);
      continue;
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if (slot < 0) continue;
    const uint32_t byte = kv8_exponent<INT8>(amax);
    const float inv = kv8_inverse(byte);
    const size_t at = kv8_row_at(p, slot, turned ? h - p.hq : h - p.hq - p.hkv);
    uint8_t* dst = (turned ? p.k_codes : p.v_codes) + at * hd;
    for (int a = 0; a < hd / 32; ++a) {
      const uint32_t code = kv8_pack4<INT8>(inv, f[a], 0.f, 0.f, 0.f);
      dst[lane + 32 * a] = static_cast<uint8_t>(byte == kv8_top<INT8>() ? kv8_below_top<INT8>(code) : code);
    }
    if (lane == 0) (turned ? p.k_exps : p.v_exps)[at] = static_cast<uint8_t>(byte);
  }
}

// ---------------------------------------------------------------- reader
constexpr int kReadThreads = 256, kReadCtas = 5;

struct Kv8ReadParams {
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const uint8_t* k_exps;
  const uint8_t* v_exps;
  __nv_bfloat16* k_out;        // [out_pages, out_size, hkv, hd]
  __nv_bfloat16* v_out;
  const int32_t* block_table;
  const int32_t* seq_lens;
  int32_t* out_table;          // [batch, out_width]
  int32_t* out_lens;           // [batch]: seq_lens within what the block table has, zero where the sequence is not read whole; or null
  int batch, hkv, log_pieces, page_size, max_pages, num_pages, out_size, out_width, out_pages;      // pieces: of 16 columns
  uint32_t inverse;            // 2^32 over the pieces of a token's row, rounded up
  ZbStatus* status;
};

ZB_DEVICE void kv8_store32(void* to, const uint32_t (&x)[8]) {      // on 32 bytes
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
               : "memory");
}

// Two codes' values times a power of two, in bf16: exact.  `from`: which bytes of a word.
template <bool INT8>
ZB_DEVICE void kv8_to_bf16(uint32_t w, float scale, uint32_t& lo, uint32_t& hi) {
  const ZbF2 by = zb_pack2(scale, scale);
  if constexpr (INT8) {
    // byte u = code + 128 in the last place of 2^23, from which the 2^23 + 128 is taken again, exactly, before the scale is multiplied: their product
    // is an infinity under scales of 2^105 and more, which rows of numbers above 2.6e33 have
    const uint32_t u = w ^ 0x80808080u;
    const ZbF2 less = zb_pack2(-8388736.f, -8388736.f);
    lo = kv8_bf16x2(zb_mul2(zb_add2(zb_pack2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441))), less), by));
    hi = kv8_bf16x2(zb_mul2(zb_add2(zb_pack2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443))), less), by));
  } else {
    uint32_t a, b;
    kv8_to_half<false>(w, a, b);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    lo = kv8_bf16x2(zb_mul2(zb_pack2(x.x, x.y), by));
    hi = kv8_bf16x2(zb_mul2(zb_pack2(y.x, y.y), by));
  }
}

// The work is a list: the pages that the sequences hold, one after another, in passes of 256 pieces of 16 columns of keys and of values; a CTA takes an
// equal, contiguous part of it, and what it writes is contiguous, too.  The sum over the sequences' pages tells which one a page belongs to, looked
// up where the page changes.  A thread has a piece of each, 16 bytes in and 32 bytes out, and asks for the next ones before it writes these.
// Bound by memory: 110000 tokens of 8 heads of 64 take 61.8 us, 5.5 TB/s (84 % of a copy's rate); 71.2 where a CTA read a head of a page at a
// time and wrote 128 bytes of every row, 64.2 with two pieces at once on four CTAs.
// SAME: pages keep their size, and a page's rows are one piece.  Else (for attention of prompts, which wants pages of 64) a thread looks every row's
// page up in the table; without SAME, pages that keep their size took 11.65 us where they take 11.1 (three sequences of up to 3300 tokens).
template <bool INT8, bool SAME>
__global__ void __launch_bounds__(kReadThreads, kReadCtas) zb_kv8_read_kernel(const Kv8ReadParams p) {
  zb_pdl_launch();
  zb_pdl_wait();
  const int most = p.max_pages * p.page_size;
  const auto pages_of = [&](int s) { return (kv8_len(p.seq_lens, s, most) + p.out_size - 1) / p.out_size; };
  const int total = kv8_total(p.batch, pages_of);
  if (total > p.out_pages && blockIdx.x == 0 && threadIdx.x == 0)
    zb_record_error(p.status, ZB_ERR_BOUNDS, kKernelKv8Read, 1u, static_cast<uint32_t>(total));
  for (int s = blockIdx.x; s < p.batch; s += gridDim.x) {
    const int first = kv8_total(s, pages_of), n = pages_of(s);
    if (p.out_lens != nullptr && threadIdx.x == 0) p.out_lens[s] = first + n <= p.out_pages ? kv8_len(p.seq_lens, s, most) : 0;
    for (int i = threadIdx.x; i < p.out_width; i += blockDim.x)
      p.out_table[static_cast<size_t>(s) * p.out_width + i] = i < n && first + i < p.out_pages ? first + i : 0;
  }
  const int per_row = p.hkv << p.log_pieces, per_page = p.out_size * per_row, passes = (per_page + kReadThreads - 1) / kReadThreads;
  const long long items = static_cast<long long>(min(total, p.out_pages)) * passes;
  const long long first = items * blockIdx.x / gridDim.x, last = items * (blockIdx.x + 1) / gridDim.x;
  if (first >= last) return;
  int left = static_cast<int>(last - first);
  int to = static_cast<int>(first / passes), pass = static_cast<int>(first - static_cast<long long>(to) * passes);
  int token0 = 0, valid = 0, page = 0;                 // the page's first token, its tokens, and what it is read from (SAME)
  const int32_t* table = nullptr;
  const auto page_of = [&](int nth) {
    const int at = table[nth];
    if (static_cast<uint32_t>(at) < static_cast<uint32_t>(p.num_pages)) return at;
    zb_record_error(p.status, ZB_ERR_BOUNDS, kKernelKv8Read, 2u, static_cast<uint32_t>(at));
    return 0;
  };
  const auto look = [&]() {
    int seq, before;
    kv8_locate(p.batch, to, pages_of, seq, before);
    token0 = (to - before) * p.out_size;
    valid = min(p.out_size, kv8_len(p.seq_lens, seq, most) - token0);
    table = p.block_table + static_cast<size_t>(seq) * p.max_pages;
    if constexpr (SAME) page = page_of(to - before);
  };
  look();
  struct Pieces {
    uint4 codes[2];
    uint32_t exps[2];
    size_t to;                                         // piece of the outputs
    bool some;                                         // the page holds it
  };
  const auto load = [&](Pieces& r) {
    const uint32_t at = pass * kReadThreads + threadIdx.x;
    r.to = static_cast<size_t>(to) * per_page + at;
    r.some = at < static_cast<uint32_t>(per_page);
    int row = __umulhi(at, p.inverse);                 // at / per_row, or one more
    row -= row * per_row > static_cast<int>(at) ? 1 : 0;
    const int rest = at - row * per_row, head = rest >> p.log_pieces, piece = rest - (head << p.log_pieces);
    const bool seen = row < valid;
    size_t from = 0;                                   // the token's row
    if (seen) {
      if constexpr (SAME) {
        from = (static_cast<size_t>(page) * p.hkv + head) * p.page_size + row;
      } else {
        const int token = token0 + row, nth = token / p.page_size;
        from = (static_cast<size_t>(page_of(nth)) * p.hkv + head) * p.page_size + (token - nth * p.page_size);
      }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      r.codes[b] = seen ? __ldcs(reinterpret_cast<const uint4*>(b ? p.v_codes : p.k_codes) + (from << p.log_pieces) + piece) : make_uint4(0u, 0u, 0u, 0u);
      r.exps[b] = seen ? (b ? p.v_exps : p.k_exps)[from] : 0u;
    }
  };
  Pieces r;
  load(r);
  while (true) {
    Pieces next = r;
    if (--left > 0) {
      if (++pass == passes) {
        pass = 0;
        ++to;
        look();
      }
      load(next);
    }
    if (r.some) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float s = kv8_scale(r.exps[b]);
        uint32_t o[8];
        kv8_to_bf16<INT8>(r.codes[b].x, s, o[0], o[1]);
        kv8_to_bf16<INT8>(r.codes[b].y, s, o[2], o[3]);
        kv8_to_bf16<INT8>(r.codes[b].z, s, o[4], o[5]);
        kv8_to_bf16<INT8>(r.codes[b].w, s, o[6], o[7]);
        kv8_store32((b ? p.v_out : p.k_out) + r.to * 16, o);
      }
    }
    if (left <= 0) return;
    r = next;
  }
}

template <int HD, int LAYOUT>
void launch_write(const Kv8WriteParams& p, bool int8, dim3 grid, int threads, cudaStream_t s) {
  if (int8) zb_launch(zb_kv8_write_kernel<HD, LAYOUT, true>, grid, dim3(threads), 0, s, p);
  else zb_launch(zb_kv8_write_kernel<HD, LAYOUT, false>, grid, dim3(threads), 0, s, p);
}
template <int LAYOUT>
void launch_write_hd(const Kv8WriteParams& p, bool int8, dim3 grid, int threads, cudaStream_t s) {
  if (p.hd == 64) launch_write<64, LAYOUT>(p, int8, grid, threads, s);
  else if (p.hd == 128) launch_write<128, LAYOUT>(p, int8, grid, threads, s);
  else launch_write<256, LAYOUT>(p, int8, grid, threads, s);
}

}  // namespace

extern "C" {

// The arguments of a call, as the caller packs them (ops/kv8.py).
struct ZbKv8Write {
  const void* qkv;
  void* q_out;
  void *k_codes, *k_exps, *v_codes, *v_exps;       // contiguous, on 16 bytes
  const int32_t* positions;
  const int32_t* slot_mapping;                     // negative: the token's keys and values are not written
  const float* inv_freq;
  const void *q_norm_w, *k_norm_w;                 // or null
  void* stream;
  long long qkv_stride, num_slots;
  int tokens, hq, hkv, hd, rot_dim, layout, page_size, norm_unit_offset, int8;
  float attn_factor, norm_eps;
};
struct ZbKv8Read {
  const void *k_codes, *k_exps, *v_codes, *v_exps;
  void *k_out, *v_out;                             // a batch that needs more is reported and read as far as they go
  const int32_t* block_table;
  const int32_t* seq_lens;
  int32_t* out_table;
  int32_t* out_lens;                               // or null
  void* stream;
  int batch, hkv, hd, page_size, max_pages, num_pages;
  int out_size, out_width, out_pages, int8;         // tokens of a page that is written, pages of a row of out_table, pages that there are
};

int zb_kv8_write(const ZbKv8Write* c) {
  if (c->tokens <= 0) return 0;
  const int hd = c->hd, rot_dim = c->rot_dim, layout = c->layout;
  if ((hd != 64 && hd != 128 && hd != 256) || rot_dim % 2 != 0 || rot_dim < 0 || rot_dim > hd || layout < 0 || layout > 2) return -42;
  if (c->page_size <= 0 || c->num_slots > 0x7fffffffll) return -43;
  ZbDeviceState* st = zb_device_state();
  if (!st) return -20;
  Kv8WriteParams p = {};
  p.qkv = reinterpret_cast<const __nv_bfloat16*>(c->qkv);
  p.q_out = reinterpret_cast<__nv_bfloat16*>(c->q_out);
  p.k_codes = reinterpret_cast<uint8_t*>(c->k_codes);
  p.v_codes = reinterpret_cast<uint8_t*>(c->v_codes);
  p.k_exps = reinterpret_cast<uint8_t*>(c->k_exps);
  p.v_exps = reinterpret_cast<uint8_t*>(c->v_exps);
  p.positions = c->positions;
  p.slot_mapping = c->slot_mapping;
  p.inv_freq = c->inv_freq;
  p.q_norm_w = reinterpret_cast<const __nv_bfloat16*>(c->q_norm_w);
  p.k_norm_w = reinterpret_cast<const __nv_bfloat16*>(c->k_norm_w);
  p.qkv_stride = c->qkv_stride;
  p.num_slots = c->num_slots;
  p.tokens = c->tokens;
  p.hq = c->hq;
  p.hkv = c->hkv;
  p.hd = hd;
  p.rot_dim = rot_dim;
  p.layout = layout;
  p.page_size = c->page_size;
  p.attn_factor = c->attn_factor;
  p.norm_eps = c->norm_eps;
  p.norm_unit_offset = c->norm_unit_offset;
  p.status = st->status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(c->stream);
  const auto at16 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; };
  const bool aligned = c->qkv_stride % 8 == 0 && at16(c->qkv) && at16(c->q_out) && at16(c->q_norm_w) && at16(c->k_norm_w);
  if (aligned && (layout == 1 || (layout == 0 && rot_dim % 16 == 0))) {
    const int units = (p.hq + 2 * p.hkv) * (hd / 16), parts = (units + 511) / 512;
    p.share = ((units + parts - 1) / parts + 31) / 32 * 32;
    const int grid = std::max(1, std::min(p.tokens, st->num_sms * std::min(1024 / p.share, 4) / parts));
    if (layout == 0) launch_write_hd<0>(p, c->int8 != 0, dim3(grid, parts), p.share, s);
    else launch_write_hd<1>(p, c->int8 != 0, dim3(grid, parts), p.share, s);
  } else if (c->int8) {
    zb_launch(zb_kv8_write_any_kernel<true>, dim3(p.tokens), dim3(256), 0, s, p);
  } else {
    zb_launch(zb_kv8_write_any_kernel<false>, dim3(p.tokens), dim3(256), 0, s, p);
  }
  zb_count_launch(1);
  return static_cast<int>(cudaGetLastError());
}

int zb_kv8_read(const ZbKv8Read* c) {
  if (c->batch <= 0) return 0;
  if (c->hd != 64 && c->hd != 128 && c->hd != 256) return -42;
  ZbDeviceState* st = zb_device_state();
  if (!st) return -20;
  Kv8ReadParams p = {};
  p.k_codes = reinterpret_cast<const uint8_t*>(c->k_codes);
  p.v_codes = reinterpret_cast<const uint8_t*>(c->v_codes);
  p.k_exps = reinterpret_cast<const uint8_t*>(c->k_exps);
  p.v_exps = reinterpret_cast<const uint8_t*>(c->v_exps);
  p.k_out = reinterpret_cast<__nv_bfloat16*>(c->k_out);
  p.v_out = reinterpret_cast<__nv_bfloat16*>(c->v_out);
  p.block_table = c->block_table;
  p.seq_lens = c->seq_lens;
  p.out_table = c->out_table;
  p.out_lens = c->out_lens;
  p.batch = c->batch;
  p.hkv = c->hkv;
  p.log_pieces = c->hd == 64 ? 2 : c->hd == 128 ? 3 : 4;
  p.page_size = c->page_size;
  p.max_pages = c->max_pages;
  p.num_pages = c->num_pages;
  p.out_size = c->out_size;
  p.out_width = c->out_width;
  p.out_pages = c->out_pages;
  p.status = st->status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(c->stream);
  const int per_row = p.hkv << p.log_pieces;
  if (static_cast<long long>(p.out_size) * per_row > 0x3fffffffll) return -43;      // pages of 16 GB
  p.inverse = static_cast<uint32_t>(((1ull << 32) + per_row - 1) / per_row);
  const long long items = static_cast<long long>(c->out_pages) * ((static_cast<long long>(p.out_size) * per_row + kReadThreads - 1) / kReadThreads);
  const dim3 grid(static_cast<unsigned>(std::max(1ll, std::min(items, static_cast<long long>(kReadCtas) * st->num_sms))));
  const bool same = c->out_size == c->page_size;
  if (same) zb_launch(c->int8 ? zb_kv8_read_kernel<true, true> : zb_kv8_read_kernel<false, true>, grid, dim3(kReadThreads), 0, s, p);
  else zb_launch(c->int8 ? zb_kv8_read_kernel<true, false> : zb_kv8_read_kernel<false, false>, grid, dim3(kReadThreads), 0, s, p);
  zb_count_launch(1);
  return static_cast<int>(cudaGetLastError());
}

}  // extern "C"
