// What the kernels of the 8-bit key / value cache share (kv8.cu: writer and reader, kv8_attention.cu: attention of single tokens).
//
// A row is one token's key or value of one head, x of HD numbers.  Its scale is the smallest power of two 2^k with max |x| <= R 2^k, R = 448
// (e4m3) and 127 (int8), and its codes are x / 2^k, which is exact, rounded to the cache's type.  A power of two costs e4m3 nothing (a floating
// format is as fine anywhere in its range) and int8 half a bit on average; in return codes times scale are bf16 numbers, so that attention over
// prompts on a bf16 copy of the cache sees the very keys and values that attention of single tokens sees, and a scale is one byte, k + 127.
// A row that holds an infinity or a NaN has the exponent byte 255 and codes of zero: it reads as NaN.  A number that would round to 2^128 takes the code below:
// what is finite reads as finite.
// Codes are [pages, kv_heads, page_size, HD], exponents [pages, kv_heads, page_size]: a page of one head is contiguous.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

// Four codes of a word -> two f16x2 (exact: e4m3 and int8 are both subsets of f16).
template <bool INT8>
ZB_DEVICE void kv8_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (INT8) {
    // byte u = code + 128 under the exponent of 1024 is 1024 + u
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));      // 1152
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias), y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

// Exponent byte of a row whose largest magnitude has the fp32 bits `amax`: exponent of R subtracted, one more where the mantissa lies above R's.
// At least 2^-100, whose reciprocal is a normal number, too.
template <bool INT8>
ZB_DEVICE uint32_t kv8_exponent(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255u;
  const int e = static_cast<int>((amax + (INT8 ? 0x01ffffu : 0x1fffffu)) >> 23) - (INT8 ? 6 : 8);
  return static_cast<uint32_t>(max(e, 27));
}
// The power of two that a byte stands for (255: infinity, which makes a NaN of the row's codes of zero; 0: zero), and its reciprocal for a row
// that is written (255: zero, so that codes are zero wherever the row has numbers).
ZB_DEVICE float kv8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
ZB_DEVICE float kv8_inverse(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }

// Four numbers of a row -> a word of codes.  `inv`: kv8_inverse of the row; where it is zero the codes are.
template <bool INT8>
ZB_DEVICE uint32_t kv8_pack4(float inv, float x0, float x1, float x2, float x3) {
  if (inv == 0.f) return 0u;
  if constexpr (INT8) {
    const uint32_t a = __byte_perm(static_cast<uint32_t>(__float2int_rn(x0 * inv)), static_cast<uint32_t>(__float2int_rn(x1 * inv)), 0x0040);
    const uint32_t b = __byte_perm(static_cast<uint32_t>(__float2int_rn(x2 * inv)), static_cast<uint32_t>(__float2int_rn(x3 * inv)), 0x0040);
    return __byte_perm(a, b, 0x5410);
  } else {
    const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(x0 * inv, x1 * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(x2 * inv, x3 * inv), __NV_SATFINITE, __NV_E4M3);
    return a | (b << 16);
  }
}
// The largest exponent byte of finite rows, under which codes of 64 (int8) or 256 (e4m3) stand for 2^128, and four of its codes with those replaced by
// the ones below, 63 and 240.  There are none above them.
template <bool INT8>
constexpr uint32_t kv8_top() { return INT8 ? 249u : 247u; }
template <bool INT8>
ZB_DEVICE uint32_t kv8_below_top(uint32_t w) {
  if constexpr (INT8) return w - (__vcmpeq4(w, 0x40404040u) & 0x01010101u) + (__vcmpeq4(w, 0xc0c0c0c0u) & 0x01010101u);
  else return w - (__vcmpeq4(w & 0x7f7f7f7fu, 0x78787878u) & 0x01010101u);
}
ZB_DEVICE uint32_t kv8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Keys of sequence `seq` as far as its block table reaches.
ZB_DEVICE int kv8_len(const int32_t* __restrict__ seq_lens, int seq, int max_keys) { return min(max(seq_lens[seq], 0), max_keys); }

// Sum of count(s) over the sequences, and the sequence whose share of that sum holds `pos` with the sum in front of it.  A warp calls
// them as a whole.
template <typename Count>
ZB_DEVICE int kv8_total(int batch, Count count) {
  int n = 0;
  for (int s = threadIdx.x & 31; s < batch; s += 32) n += count(s);
  return __reduce_add_sync(0xffffffffu, n);
}
template <typename Count>
ZB_DEVICE void kv8_locate(int batch, int pos, Count count, int& seq, int& before) {
  const int lane = threadIdx.x & 31;
  before = 0;
  for (int s0 = 0; s0 < batch; s0 += 32) {
    const int n = s0 + lane < batch ? count(s0 + lane) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + upto > pos);
    if (past != 0u) {
      const int at = __ffs(past) - 1;
      seq = s0 + at;
      before += __shfl_sync(0xffffffffu, upto - n, at);
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  seq = batch;      // pos lies behind the last sequence
}
