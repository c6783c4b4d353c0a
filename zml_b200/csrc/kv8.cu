// Writer and reader of the paged key / value cache in 8 bits (format: kv8.cuh).
//
//   zb_kv8_write   one pass over the fused projection [T, (Hq + 2 Hkv) * HD]: optional RMSNorm of every query and key head, rotation by
//                  the token's position, queries to bf16, keys and values to codes and exponents at their slots
//   zb_kv8_read    whole sequences out of their pages into dense bf16 pages [pages, page_size, Hkv, HD], and the block table of those
//
// Between the bf16 projection and the one rounding at the end (bf16 queries, codes) everything is fp32: a rounding to bf16 in between would put
// three codes of a hundred into the neighbouring step.  Angles p * f are formed and reduced in fp64 (one per pair of columns and token, used
// by all heads), so that far positions keep the digits that fp32 products lose (1e5 radians: 0.004).
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

// cos and sin of position * frequency, both within about 1.5 ulp of fp32.
ZB_DEVICE void kv8_angle(int pos, float freq, float factor, float& sn, float& cs) {
  const double a = static_cast<double>(pos) * static_cast<double>(freq);
  const double r = fma(-rint(a * 0.15915494309189535), 6.283185307179586, a);
  const float hi = static_cast<float>(r), lo = static_cast<float>(r - static_cast<double>(hi));
  float s, c;
  sincosf(hi, &s, &c);
  sn = fmaf(c, lo, s) * factor;
  cs = fmaf(-s, lo, c) * factor;
}

// Slot of token `tok`: -1 for a token that writes nothing.  One behind the cache is reported.
ZB_DEVICE long long kv8_slot(const Kv8WriteParams& p, int tok) {
  const long long slot = p.slot_mapping[tok];
  if (slot >= p.num_slots) {
    if (threadIdx.x == 0) zb_record_error(p.status, ZB_ERR_BOUNDS, kKernelKv8Write, 1u, static_cast<uint32_t>(slot));
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
// eight columns of one head: the two that rotate into each other, or two neighbours.  The HD / 16 threads of a head lie in one warp and add up
// its squares and its largest magnitude.  One CTA takes a token (few tokens of many heads: a part of its pieces).
template <int HD, int LAYOUT, bool INT8>
__global__ void __launch_bounds__(512) zb_kv8_write_kernel(const Kv8WriteParams p) {
  constexpr int kLanes = HD / 16;
  __shared__ __align__(16) float sn[HD / 2], cs[HD / 2];
  zb_pdl_launch();
  zb_pdl_wait();
  const int tok = blockIdx.x, half = p.rot_dim >> 1;
  const int pos = p.positions[tok];
  const long long slot = kv8_slot(p, tok);
  const int from = static_cast<int>(blockIdx.y) * p.share, units = min(from + p.share, (p.hq + 2 * p.hkv) * kLanes);
  const int rounded = from + ((units - from + 31) & ~31);      // a warp goes through the loop as a whole
  bool first = true;
  for (int u0 = from + threadIdx.x; u0 < rounded; u0 += blockDim.x) {
    const bool in = u0 < units;
    const int u = in ? u0 : units - 1, h = u / kLanes, j = u - h * kLanes;
    const bool is_q = h < p.hq, turned = h < p.hq + p.hkv;
    const bool turns = LAYOUT == 0 && turned && j < half / 8;
    // 8-column pieces of the head
    const int a0 = LAYOUT == 1 || !turned ? 2 * j : (turns ? j : half / 4 + 2 * (j - half / 8));
    const int a1 = turns ? j + half / 8 : a0 + 1;
    const uint4* src = reinterpret_cast<const uint4*>(p.qkv + static_cast<size_t>(tok) * p.qkv_stride + static_cast<size_t>(h) * HD);
    const uint4 x0 = src[a0], x1 = src[a1];
    if (first) {                                     // the angles, while the loads are on their way
      first = false;
      for (int i = threadIdx.x; i < half; i += blockDim.x) kv8_angle(pos, p.inv_freq[i], p.attn_factor, sn[i], cs[i]);
      __syncthreads();
    }
    float f0[8], f1[8];
    kv8_unpack8(x0, f0);
    kv8_unpack8(x1, f1);
    const uint32_t group = ((1ull << kLanes) - 1ull) << ((threadIdx.x & 31) / kLanes * kLanes);
    if (turned) {
      const __nv_bfloat16* nw = is_q ? p.q_norm_w : p.k_norm_w;
      if (nw != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += f0[i] * f0[i] + f1[i] * f1[i];
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
        const float inv = rsqrtf(ss / static_cast<float>(HD) + p.norm_eps), one = p.norm_unit_offset ? 1.f : 0.f;
        float g0[8], g1[8];
        kv8_unpack8(reinterpret_cast<const uint4*>(nw)[a0], g0);
        kv8_unpack8(reinterpret_cast<const uint4*>(nw)[a1], g1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          f0[i] = f0[i] * inv * (g0[i] + one);
          f1[i] = f1[i] * inv * (g1[i] + one);
        }
      }
      if (LAYOUT == 0) {
        if (turns) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float c_ = cs[8 * j + i], s_ = sn[8 * j + i], x = f0[i], y = f1[i];
            f0[i] = x * c_ - y * s_;
            f1[i] = y * c_ + x * s_;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int i0 = 8 * j + i, i1 = i0 + 4;
          if (i0 < half) {
            const float x = f0[2 * i], y = f0[2 * i + 1];
            f0[2 * i] = x * cs[i0] - y * sn[i0];
            f0[2 * i + 1] = y * cs[i0] + x * sn[i0];
          }
          if (i1 < half) {
            const float x = f1[2 * i], y = f1[2 * i + 1];
            f1[2 * i] = x * cs[i1] - y * sn[i1];
            f1[2 * i + 1] = y * cs[i1] + x * sn[i1];
          }
        }
      }
    }
    if (is_q) {
      if (!in) continue;
      uint4* dst = reinterpret_cast<uint4*>(p.q_out + (static_cast<size_t>(tok) * p.hq + h) * HD);
      dst[a0] = make_uint4(zb_pack_bf16x2(f0[0], f0[1]), zb_pack_bf16x2(f0[2], f0[3]), zb_pack_bf16x2(f0[4], f0[5]), zb_pack_bf16x2(f0[6], f0[7]));
      dst[a1] = make_uint4(zb_pack_bf16x2(f1[0], f1[1]), zb_pack_bf16x2(f1[2], f1[3]), zb_pack_bf16x2(f1[4], f1[5]), zb_pack_bf16x2(f1[6], f1[7]));
      continue;
    }
    uint32_t amax = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, max(kv8_abs_bits(f0[i]), kv8_abs_bits(f1[i])));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(group, amax, o));
    if (!in || slot < 0) continue;
    const uint32_t byte = kv8_exponent<INT8>(amax);
    const float inv = kv8_inverse(byte);
    const int kvh = turned ? h - p.hq : h - p.hq - p.hkv;
    const size_t at = kv8_row_at(p, slot, kvh);
    uint2* dst = reinterpret_cast<uint2*>((turned ? p.k_codes : p.v_codes) + at * HD);
    dst[a0] = make_uint2(kv8_pack4<INT8>(inv, f0[0], f0[1], f0[2], f0[3]), kv8_pack4<INT8>(inv, f0[4], f0[5], f0[6], f0[7]));
    dst[a1] = make_uint2(kv8_pack4<INT8>(inv, f1[0], f1[1], f1[2], f1[3]), kv8_pack4<INT8>(inv, f1[4], f1[5], f1[6], f1[7]));
    if (j == 0) (turned ? p.k_exps : p.v_exps)[at] = static_cast<uint8_t>(byte);
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
    for (int a = 0; a < hd / 32; ++a) dst[lane + 32 * a] = static_cast<uint8_t>(kv8_pack4<INT8>(inv, f[a], 0.f, 0.f, 0.f));
    if (lane == 0) (turned ? p.k_exps : p.v_exps)[at] = static_cast<uint8_t>(byte);
  }
}

// ---------------------------------------------------------------- reader
struct Kv8ReadParams {
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const uint8_t* k_exps;
  const uint8_t* v_exps;
  __nv_bfloat16* k_out;        // [out_pages, page_size, hkv, hd]
  __nv_bfloat16* v_out;
  const int32_t* block_table;
  const int32_t* seq_lens;
  int32_t* out_table;          // [batch, max_pages]
  int batch, hkv, page_size, max_pages, num_pages, out_pages;
  ZbStatus* status;
};

// A CTA takes (page, keys or values, head) after (page, ...) of all pages that the sequences hold; the sum over the sequences' pages tells
// which one a page belongs to.  A thread has eight codes of a row: 8 bytes in, 16 bytes out.
template <int HD, bool INT8>
__global__ void __launch_bounds__(256) zb_kv8_read_kernel(const Kv8ReadParams p) {
  constexpr int kPieces = HD / 8;
  zb_pdl_launch();
  zb_pdl_wait();
  const auto pages_of = [&](int s) { return (kv8_len(p.seq_lens, s, p.max_pages * p.page_size) + p.page_size - 1) / p.page_size; };
  const int total = kv8_total(p.batch, pages_of), items = min(total, p.out_pages) * 2 * p.hkv;
  if (total > p.out_pages && blockIdx.x == 0 && threadIdx.x == 0)
    zb_record_error(p.status, ZB_ERR_BOUNDS, kKernelKv8Read, 1u, static_cast<uint32_t>(total));
  for (int s = blockIdx.x; s < p.batch; s += gridDim.x) {
    const int first = kv8_total(s, pages_of), n = pages_of(s);
    for (int i = threadIdx.x; i < p.max_pages; i += blockDim.x)
      p.out_table[static_cast<size_t>(s) * p.max_pages + i] = i < n && first + i < p.out_pages ? first + i : 0;
  }
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int to = item / (2 * p.hkv), rest = item - to * 2 * p.hkv, kv = rest / p.hkv, head = rest - kv * p.hkv;
    int seq, before;
    kv8_locate(p.batch, to, pages_of, seq, before);
    const int nth = to - before, valid = min(p.page_size, kv8_len(p.seq_lens, seq, p.max_pages * p.page_size) - nth * p.page_size);
    int page = p.block_table[static_cast<size_t>(seq) * p.max_pages + nth];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.num_pages)) {
      if (threadIdx.x == 0) zb_record_error(p.status, ZB_ERR_BOUNDS, kKernelKv8Read, 2u, static_cast<uint32_t>(page));
      page = 0;
    }
    const size_t from = (static_cast<size_t>(page) * p.hkv + head) * p.page_size;
    const uint2* src = reinterpret_cast<const uint2*>((kv ? p.v_codes : p.k_codes) + from * HD);
    const uint8_t* ex = (kv ? p.v_exps : p.k_exps) + from;
    __nv_bfloat16* dst = (kv ? p.v_out : p.k_out) + (static_cast<size_t>(to) * p.page_size * p.hkv + head) * HD;
#pragma unroll 4
    for (int i = threadIdx.x; i < p.page_size * kPieces; i += 256) {
      const int row = i / kPieces, piece = i - row * kPieces;
      uint4 o = make_uint4(0u, 0u, 0u, 0u);
      if (row < valid) {
        const uint2 w = src[i];
        const float s = kv8_scale(ex[row]);
        uint32_t h[4], b[4];
        kv8_to_half<INT8>(w.x, h[0], h[1]);
        kv8_to_half<INT8>(w.y, h[2], h[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
          b[e] = zb_pack_bf16x2(v.x * s, v.y * s);
        }
        o = make_uint4(b[0], b[1], b[2], b[3]);
      }
      *reinterpret_cast<uint4*>(dst + static_cast<size_t>(row) * p.hkv * HD + piece * 8) = o;
    }
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
  void *k_out, *v_out;                             // out_pages pages; a batch that needs more is reported and read as far as they go
  const int32_t* block_table;
  const int32_t* seq_lens;
  int32_t* out_table;
  void* stream;
  int batch, hkv, hd, page_size, max_pages, num_pages, out_pages, int8;
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
    const int units = (p.hq + 2 * p.hkv) * (hd / 16), parts = p.tokens <= 64 ? (units + 511) / 512 : 1;
    p.share = ((units + parts - 1) / parts + 31) / 32 * 32;
    const int threads = p.share < 512 ? p.share : 512;
    if (layout == 0) launch_write_hd<0>(p, c->int8 != 0, dim3(p.tokens, parts), threads, s);
    else launch_write_hd<1>(p, c->int8 != 0, dim3(p.tokens, parts), threads, s);
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
  p.batch = c->batch;
  p.hkv = c->hkv;
  p.page_size = c->page_size;
  p.max_pages = c->max_pages;
  p.num_pages = c->num_pages;
  p.out_pages = c->out_pages;
  p.status = st->status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(c->stream);
  const long long items = static_cast<long long>(c->out_pages) * 2 * c->hkv;
  if (items > 0x7fffffffll) return -43;
  const int most = st->num_sms * 8;
  const dim3 grid(static_cast<unsigned>(items < 1 ? 1 : (items < most ? items : most)));
  const bool int8 = c->int8 != 0;
  if (c->hd == 64) zb_launch(int8 ? zb_kv8_read_kernel<64, true> : zb_kv8_read_kernel<64, false>, grid, dim3(256), 0, s, p);
  else if (c->hd == 128) zb_launch(int8 ? zb_kv8_read_kernel<128, true> : zb_kv8_read_kernel<128, false>, grid, dim3(256), 0, s, p);
  else zb_launch(int8 ? zb_kv8_read_kernel<256, true> : zb_kv8_read_kernel<256, false>, grid, dim3(256), 0, s, p);
  zb_count_launch(1);
  return static_cast<int>(cudaGetLastError());
}

}  // extern "C"
