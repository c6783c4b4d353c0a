// The draw of one token for each row of logits, with temperature, top-k, top-p and min-p of every row, from given random numbers.
//
// With M = max x, w_i = 2^((x_i - M) log2(e) / T): the top_k largest stay (equal ones: the lower indices); of these, in the order of their size, those
// whose predecessors' weights are less than top_p of the sum; of these, those with w_i >= min_p.  The token is the first in the vocabulary's order up to which the
// weights that stayed sum to more than u times their sum.
//
// Weights are whole numbers of 2^-44 of the largest, so that sums of a whole row are exact in 64 bits and do not depend on an order.  A weight is off by 2^-45 and, its
// logarithm having 41 bits behind the point, by 2^-42 of itself; a sum of n by n 2^-45 and 2^-42 of itself at most.  (A sum of fp32 weights is off by 1e-7 of the whole, and among 128 thousand flat weights each is 8e-6 of it:
// one draw in a hundred would be another token.)
//
// A cluster of CTAs has a row, a slice a CTA, and reads it two to four times, all but the first time from L2 (shared memory for the slices would leave two
// CTAs on an SM: 64 rows of 151936 40 us, 256 380).  The row is not sorted.  All cuts keep what is in front in the order of size, so a row ends in one of two ways:
//   * a list: what is at least as large as a bound - the k-th largest of some logits; the weight below which all of the vocabulary together is less than
//     1 - top_p; the end of the bin of a histogram in which the cut is - is usually a few hundred logits, which one CTA ranks, sums and draws from;
//   * a cut: where these are too many, one more pass sums the weights above the histogram's bins that may have the cut and lists what is in them, 11 bits of
//     a logit at a time tell which of these is the smallest that stays and how many of its equals do, and the warp that has the drawn one looks for it.
// The histogram has a bin for each 2^-9 .. 2^-4 of the weights' logarithm and counts logits, in the pass that sums all weights; a bin's edges bound the weights in it (a
// histogram over the logits after that pass, with the weights of each bin's middle, and a list tried beforehand: 256 rows with flat logits 322 us, now 257).
// What bounds it: the passes over many rows, whose instructions are some 30 of a weight and some 40 with the histogram's, and some 120 an element in all for a wide nucleus;
// for few rows the passes' and the cluster's barriers' latency.  Measured: 1 row of 128256 with top_p 15 us, 32 rows with settings of their own 32 - 43 by the settings
// that were drawn, 64 rows of 151936 without a cut 36, 128 rows of 248320 with top_k 50 and top_p 55 (127 MB: 2.3 TB/s), 256 rows of 151936 with a nucleus of 80 thousand 259.
// (A small top_k alone: the library's kernel for up to 128 candidates, which ranks and draws with noise, takes 10 us for a row of 128256 where this one takes 13.)
#include <algorithm>

#include "common.cuh"
#include "host_api.h"

namespace {

constexpr int kMaxCtas = 8;
constexpr int kMaxVocab = 8 * 49152;                 // (an index and a weight are one number of 19 + 45 bits)
constexpr int kList = 2048;
// A top_k up to this ends in a list, if all goes well.  Rows alike, top_k 1000, by lists and by cuts, us: 1 x 32000 17 / 22, 1 x 248320 24 / 36, 32 x 128256 33 / 47, 256 x 128256
// 140 / 177; top_k 601: 14 / 21, 21 / 35, 29 / 47, 109 / 164.  Beyond it the lists of 2048 overflow: a top_k of 1500 that tries one first takes 31 / 23, 54 / 38, 68 / 48, 268 / 189.
constexpr int kSmallK = 1024;
constexpr int kBins = 2048;
constexpr int kTable = 16;                           // 2^((j + 1/2) / 16): any 32 lanes' entries are on different banks (512 entries: 7 conflicts)
constexpr double kOne = 17592186044416.0;            // 2^44
constexpr double kMiddle = 1.5 * 2048.0;             // a number of less than 1024, added to it, has its 2^-41 in the last place
constexpr unsigned long long kBias = 0x4070000000000000ull;      // 256.0: a weight added to it has its 2^-44 in the last place

struct SampleParams {
  const void* logits;
  int32_t* token;
  float* logprob;
  const void* uniforms;          // fp32 or fp64, or null: rng
  const unsigned long long* rng; // {seed, draws so far}
  const float *temperature, *top_p, *min_p;      // per row, or null: the numbers below
  const int32_t* top_k;
  long long stride;
  double temperature_all, top_p_all, min_p_all;
  int top_k_all, vocab, uniforms64, vec;         // vec: every row starts on four logits
  int slice, filled;             // slice: of a CTA, whole rows of 128 for each warp; filled: CTAs of which three quarters or more have logits (at least one)
};

using u64 = unsigned long long;

// Order-preserving; one zero.  NaN does not come here.
ZB_DEVICE uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
ZB_DEVICE float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

ZB_DEVICE double uniform53(u64 seed, u64 draw, int row) {
  // splitmix64 of (seed, draw, row)
  uint64_t z = seed + 0x9e3779b97f4a7c15ull * (draw * 0x100000000ull + static_cast<uint64_t>(row) + 1);
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  z ^= z >> 31;
  return static_cast<double>(z >> 11) * 0x1p-53;
}

ZB_DEVICE void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
ZB_DEVICE void st_cluster_u64(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
ZB_DEVICE u64 ld_cluster_u64(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
ZB_DEVICE uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
ZB_DEVICE void cluster_sync() {
  zb_cluster_arrive();
  zb_cluster_wait();
}
ZB_DEVICE u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
ZB_DEVICE u64 warp_upto(u64 v, int lane) {           // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <int kThreads>
struct Shared {
  static constexpr int kWarps = kThreads / 32;
  double table[kTable];
  u64 cand[kList];                                   // of this CTA: key << 32 | ~index, the larger, the further in front
  union {
    u64 sorted[kList];                               // CTA 0: of the cluster
    uint32_t hist[kBins];
  };
  union {
    u64 weight[kList];                               // CTA 0: of these; then those that stay, index << 45 | weight
    u64 sums[kBins];
  };
  u64 part[kWarps], seg[kWarps], sub[kWarps], above[kWarps];
  u64 total[kMaxCtas], lower[kMaxCtas];              // of every CTA
  uint32_t ties[kMaxCtas], count[kMaxCtas], best[kMaxCtas], bound[kMaxCtas], least[kMaxCtas];
  uint32_t seg_ties[kWarps], sub_ties[kWarps], warp_best[kWarps], warp_least[kWarps], top[kThreads], n, range[2];
  u64 left;                                          // what one thread of the cluster has found, in every CTA
  uint32_t found[3];
};

// All threads of a cluster, which is one row.
template <typename T, int kThreads>
struct Sampler {
  static constexpr int kWarps = kThreads / 32, kMine = kList / kThreads;      // neighbours of a list that a thread has
  const SampleParams& p;
  Shared<kThreads>& sh;
  const T* x;                    // the row
  int ctas, rank, warp, lane, from, end;              // the warp's part of the row, whole rows of 128 but for the row's end
  int kind;                      // 1: only infinities count, as 1; 2: logits are scaled by 2^-64
  float top, floor_x;            // the largest logit; below floor_x weights are zero
  double top64, scale;           // log2 of a weight is (x - top) * scale
  uint32_t best;
  int bin_from, bin_shift;       // see count_bins
  bool listed;                   // the logits around the cut are in the CTAs' lists, and what is above them in sh.above

  ZB_DEVICE Sampler(const SampleParams& params, Shared<kThreads>& shared, int log2_ctas)
      : p(params), sh(shared), ctas(1 << log2_ctas), rank(blockIdx.x & (ctas - 1)), warp(threadIdx.x >> 5), lane(threadIdx.x & 31), kind(0), listed(false) {
    x = reinterpret_cast<const T*>(p.logits) + static_cast<size_t>(blockIdx.x >> log2_ctas) * p.stride;
    from = min(rank * p.slice + warp * (p.slice / kWarps), p.vocab);
    end = min(from + p.slice / kWarps, p.vocab);
  }

  // The weight of a logit that is not above `top`, in 2^-44, plus kBias; a NaN's is zero.  z is held with 41 bits behind the point: 4 of them choose the table's
  // entry, and with the other 37 as r, around their middle, 2^r is a polynomial (off by 5e-16).
  ZB_DEVICE double log2_of(float x) const { return __fma_rn(static_cast<double>(fmaxf(x, floor_x)) - top64, scale, kMiddle); }
  ZB_DEVICE u64 biased(float x) const { return power(log2_of(x)); }
  ZB_DEVICE u64 power(double t) const {
    const int hi = __double2hiint(t);
    const double r = __hiloint2double(0x43300000 | (hi & 31), __double2loint(t)) - 4503668346847232.0;      // 2^52 + 2^36
    constexpr double c1 = 0.6931471805599453 * 0x1p-41, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4, c5 = c4 * c1 / 5, c6 = c5 * c1 / 6;
    const double base = sh.table[hi >> 5 & (kTable - 1)];
    const double b = __hiloint2double(__double2hiint(base) + ((hi & ~0x1ff) << 11) - (1024 << 20), __double2loint(base));
    const double q = __fma_rn(__fma_rn(__fma_rn(__fma_rn(__fma_rn(r, c6, c5), r, c4), r, c3), r, c2), r, c1) * r;
    return static_cast<u64>(__double_as_longlong(__fma_rn(b, q, b) + 256.0));
  }
  ZB_DEVICE u64 weight(float x) const { return biased(x) - kBias; }

  ZB_DEVICE float fix(float v) const {               // what counts as a logit (a NaN fails every comparison and has no weight)
    return kind == 0 ? v : kind == 1 ? (v == INFINITY ? 1.f : -INFINITY) : v * 0x1p-64f;
  }
  // f(four logits, index of the first, distance of their indices) over the warp's part, 128 logits at a time, -inf behind the row's end.
  template <typename F>
  ZB_DEVICE void each(F&& f) const {
    constexpr int kOnce = 4;
    int i = from;
    if (p.vec) {
#pragma unroll 1
      for (; i + 128 <= end; i += 128 * kOnce) {
        float4 v[kOnce];
#pragma unroll
        for (int k = 0; k < kOnce; ++k) {
          const int at = i + k * 128 + lane * 4;
          if (i + (k + 1) * 128 <= end) {
            if constexpr (sizeof(T) == 4) {
              v[k] = *reinterpret_cast<const float4*>(x + at);
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(x + at);
              v[k] = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
            }
          }
        }
#pragma unroll
        for (int k = 0; k < kOnce; ++k) {
          if (i + (k + 1) * 128 > end) break;
          float e[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          if (kind != 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = fix(e[j]);
          }
          f(e, i + k * 128 + lane * 4, 1);
        }
      }
      i = from + (end - from) / 128 * 128;
    }
#pragma unroll 1
    for (; i < end; i += 128) {
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = i + j * 32 + lane;
        e[j] = at < end ? fix(static_cast<float>(x[at])) : -INFINITY;
      }
      f(e, i + lane, 32);
    }
  }

  // The k-th largest of at least k of the CTA's logits (at most 32 a warp): each warp's largest few of its lanes' largest.
  ZB_DEVICE void find_bound(uint32_t mine, int k) {
    const int share = (k + kWarps - 1) / kWarps, per_warp = min(share + share / 2 + 1, 32);      // (half as many again, so that the k-th is not just the worst warp's last)
    for (int i = 0; i < per_warp; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, mine);
      const uint32_t who = __ballot_sync(0xffffffffu, mine == m);
      if (lane == __ffs(who) - 1) mine = 0;
      if (lane == 0) sh.top[i * kWarps + warp] = m;
    }
    __syncthreads();
    if (threadIdx.x < kWarps * per_warp) {
      const uint32_t m = sh.top[threadIdx.x];
      int ahead = 0;
#pragma unroll 4
      for (int j = 0; j < kWarps * per_warp; ++j) ahead += sh.top[j] > m || (sh.top[j] == m && j < static_cast<int>(threadIdx.x)) ? 1 : 0;
      if (ahead == k - 1) sh.range[0] = m;
    }
    __syncthreads();
  }

  // Over the cluster, in every thread.  (Another barrier has to come before the next sum.)
  ZB_DEVICE u64 sum_all(u64 v) {
    v = warp_sum(v);
    if (lane == 0) sh.part[warp] = v;
    __syncthreads();
    if (warp == 0) {
      u64 s = lane < kWarps ? sh.part[lane] : 0;
      s = warp_sum(s);
      if (lane < ctas) st_cluster_u64(zb_mapa(zb_smem_u32(&sh.total[rank]), lane), s);
    }
    cluster_sync();
    u64 s = 0;
    for (int c = 0; c < ctas; ++c) s += sh.total[c];
    return s;
  }

  // Four of a lane's logits into the CTA's list, by whole warps.
  ZB_DEVICE void append(const bool (&some)[4], const float (&v)[4], int index, int step) {
    uint32_t who[4];
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) who[j] = __ballot_sync(0xffffffffu, some[j]), n += __popc(who[j]);
    if (n == 0) return;
    uint32_t slot = 0;
    if (lane == 0) slot = atomicAdd(&sh.n, static_cast<uint32_t>(n));
    slot = __shfl_sync(0xffffffffu, slot, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t mine = slot + __popc(who[j] & ((1u << lane) - 1u));
      if (some[j] && mine < kList) sh.cand[mine] = static_cast<u64>(key_of(v[j])) << 32 | static_cast<uint32_t>(~(index + j * step));
      slot += __popc(who[j]);
    }
  }
  // Every CTA's sh.n to all; how many in the cluster, more than kList: too many.
  ZB_DEVICE int exchange_counts() {
    __syncthreads();
    if (threadIdx.x < ctas) st_cluster_u32(zb_mapa(zb_smem_u32(&sh.count[rank]), threadIdx.x), sh.n);
    cluster_sync();
    int n = 0;
    for (int c = 0; c < ctas; ++c) n += static_cast<int>(min(sh.count[c], static_cast<uint32_t>(kList + 1)));
    return n;
  }
  // A row's logits from key `lo` on into the CTAs' lists; how many.  (Another barrier has to come before the lists are written again.)
  ZB_DEVICE int gather(uint32_t lo) {
    const float bound = value_of(lo);
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    const volatile uint32_t* n = &sh.n;
    each([&](const float (&e)[4], int at, int step) {
      if (!__any_sync(0xffffffffu, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])) >= bound)) return;
      if (__shfl_sync(0xffffffffu, *n, 0) > kList) return;      // too many already
      bool in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) in[j] = e[j] >= bound && at + j * step < end;
      append(in, e, at, step);
    });
    return exchange_counts();
  }

  // The CTAs' lists, n in all, of keys from `least` on, to CTA 0, in the order of size.
  ZB_DEVICE void sort_lists(int n, uint32_t least) {
    if (rank == 0) {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        int c = 0, at = i;
        while (at >= static_cast<int>(sh.count[c])) at -= sh.count[c++];
        sh.sorted[i] = ld_cluster_u64(zb_mapa(zb_smem_u32(&sh.cand[at]), c));
      }
    }
    cluster_sync();                                  // nobody leaves or writes its list before it has been read
    if (rank == 0) sort_down(sh.sorted, sh.weight, n, static_cast<u64>(least) << 32, static_cast<u64>(best) << 32 | 0xffffffffu);
  }
  // a[0, n), of numbers in [lo, hi] and no two alike, from the largest on, by counting what is in front of each: of all, or (1016: 3 us, bitonically 12) of an interval of 2048.
  // b, sh.cand: space.
  ZB_DEVICE void sort_down(u64* a, u64* b, int n, u64 lo, u64 hi) {
    __syncthreads();
    if (n <= min(kThreads, 256)) {
      int ahead = 0;
      u64 mine = 0;
      if (static_cast<int>(threadIdx.x) < n) {
        mine = a[threadIdx.x];
#pragma unroll 8
        for (int j = 0; j < n; ++j) ahead += a[j] > mine ? 1 : 0;
      }
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < n) a[ahead] = mine;
      __syncthreads();
      return;
    }
    constexpr int kOwn = kBins / kThreads;
    uint32_t* ends = reinterpret_cast<uint32_t*>(sh.cand) + 1;      // of the intervals, from the highest on: ends[-1] is 0
    const int shift = max(0, 53 - __clzll(static_cast<long long>(hi - lo)));
    const auto interval = [&](u64 v) { return static_cast<int>((hi - v) >> shift); };
    for (int i = threadIdx.x; i <= kBins; i += kThreads) ends[i - 1] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) atomicAdd(&ends[interval(a[i])], 1u);
    __syncthreads();
    uint32_t count[kOwn], mine = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) mine += count[j] = ends[threadIdx.x * kOwn + j];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) sh.seg_ties[warp] = upto;
    __syncthreads();
    upto -= mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) upto += w < warp ? sh.seg_ties[w] : 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      ends[threadIdx.x * kOwn + j] = upto;           // where it begins, until its numbers are there
      upto += count[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) b[atomicAdd(&ends[interval(a[i])], 1u)] = a[i];
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const u64 v = b[i];
      const int at = interval(v), first = ends[at - 1], last = ends[at];
      int ahead = first;
      for (int j = first; j < last; ++j) ahead += b[j] > v ? 1 : 0;
      a[ahead] = v;
    }
    __syncthreads();
  }
  static ZB_DEVICE uint32_t key_at(u64 c) { return static_cast<uint32_t>(c >> 32); }
  static ZB_DEVICE int index_at(u64 c) { return ~static_cast<int>(static_cast<uint32_t>(c)); }

  // Given their weights: what is in front of the first; *all: the sum of the list.
  ZB_DEVICE u64 list_before(const u64 (&w)[kMine], u64* all) {
    u64 mine = 0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) mine += w[j];
    const u64 upto = warp_upto(mine, lane);
    if (lane == 31) sh.part[warp] = upto;
    __syncthreads();
    u64 before = upto - mine;
    *all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const u64 y = sh.part[i];
      if (i < warp) before += y;
      *all += y;
    }
    __syncthreads();
    return before;
  }

  ZB_DEVICE double uniform(int row) const {
    double u;
    if (p.uniforms == nullptr) u = uniform53(p.rng[0], p.rng[1], row);
    else u = p.uniforms64 ? reinterpret_cast<const double*>(p.uniforms)[row] : static_cast<double>(reinterpret_cast<const float*>(p.uniforms)[row]);
    return u > 0.0 ? fmin(u, 1.0) : 0.0;             // NaN: 0
  }
  static ZB_DEVICE u64 target_of(double u, u64 all) { return min(static_cast<u64>(u * static_cast<double>(all)), all - 1); }
  static ZB_DEVICE u64 need_of(double top_p, u64 all) { return min(max(1ull, static_cast<u64>(ceil(top_p * static_cast<double>(all)))), all); }
  ZB_DEVICE void write(int row, int token, float x, u64 all) const {
    p.token[row] = token;
    if (p.logprob != nullptr)
      p.logprob[row] = static_cast<float>((static_cast<double>(x) - top64) * scale * 0.6931471805599453 - log(static_cast<double>(all) / kOne));
  }

  // CTA 0: from the sorted list of n, of which those with keys from `least` on may stay; `all`: the sum that top_p is a part of, 0: the list's.
  ZB_DEVICE void draw_from_list(int row, int n, double top_p, u64 all, uint32_t least) {
    const int i = kMine * threadIdx.x;
    u64 c[kMine], w[kMine], sum;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      c[j] = i + j < n ? sh.sorted[i + j] : 0;
      w[j] = i + j < n ? weight(value_of(key_at(c[j]))) : 0;
    }
    u64 before = list_before(w, &sum);
    const u64 need = top_p < 1.0 ? need_of(top_p, all != 0 ? all : sum) : ~0ull;
    int stays = 0;                                   // the first few of the list
    u64 kept = 0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      if (i + j < n && (i + j == 0 || (before < need && key_at(c[j]) >= least))) {
        ++stays;
        kept += w[j];
        sh.weight[i + j] = static_cast<u64>(static_cast<uint32_t>(0x7ffffu - index_at(c[j]))) << 45 | w[j];      // (sorted down: the lowest index first)
      }
      before += w[j];
    }
    int m = __reduce_add_sync(0xffffffffu, stays);
    kept = warp_sum(kept);
    if (lane == 0) sh.sub[warp] = kept, sh.sub_ties[warp] = m;
    __syncthreads();
    m = 0, kept = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) m += sh.sub_ties[k], kept += sh.sub[k];
    const u64 target = target_of(uniform(row), kept);
    constexpr u64 kWeight = (1ull << 45) - 1;
    const auto found = [&](u64 number) {
      const int token = 0x7ffff - static_cast<int>(number >> 45);
      write(row, token, fix(static_cast<float>(x[token])), kept);
    };
    if (m <= min(kThreads, 256)) {
      if (static_cast<int>(threadIdx.x) >= m) return;
      const u64 mine = sh.weight[threadIdx.x];
      before = 0;
#pragma unroll 8
      for (int j = 0; j < m; ++j) {
        const u64 y = sh.weight[j];
        before += y > mine ? y & kWeight : 0;        // (of lower index; no two have the same)
      }
      if (before <= target && target - before < (mine & kWeight)) found(mine);
      return;
    }
    sort_down(sh.weight, sh.sorted, m, static_cast<u64>(0x80000 - p.vocab) << 45, (1ull << 63) + ((1ull << 63) - 1));
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      c[j] = i + j < m ? sh.weight[i + j] : 0;
      w[j] = c[j] & kWeight;
    }
    before = list_before(w, &sum);
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      if (before <= target && target - before < w[j]) found(c[j]);
      before += w[j];
    }
  }

  // ---- the cuts of rows that are too long for a list
  // Counts of the logits with weights of 2^z_from or more, in up to 2048 bins of equal length on the weights' logarithm (the high word of log2_of: 2^-9 or
  // more; from the row's smallest logit on).  With `list` they are listed, too, until there are too many.  Returns the thread's sum of weights.
  ZB_DEVICE u64 count_bins(double z_from, uint32_t row_least, bool sums, bool list) {
    bin_from = max(__double2hiint(log2_of(value_of(row_least))), __double2hiint(kMiddle + z_from));
    bin_shift = max(0, 21 - __clz(__double2hiint(kMiddle) - bin_from));
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = 0;
    if (threadIdx.x == 0) sh.n = list ? 0 : kList + 1;
    __syncthreads();
    u64 sum = 0;
    uint32_t counted = 0;
    const volatile uint32_t* listed_so_far = &sh.n;
    each([&](const float (&e)[4], int at, int step) {
      int d[4], most = -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double t = log2_of(e[j]);
        if (sums) sum += power(t);
        d[j] = __double2hiint(t) - bin_from;
        most = max(most, d[j]);
      }
      counted += 4;
      if (!__any_sync(0xffffffffu, most >= 0)) return;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d[j] >= 0) atomicAdd(&sh.hist[d[j] >> bin_shift], 1u);
      if (list) {
        if (__shfl_sync(0xffffffffu, *listed_so_far, 0) > kList) list = false;
        const bool in[4] = {d[0] >= 0, d[1] >= 0, d[2] >= 0, d[3] >= 0};
        append(in, e, at, step);
      }
    });
    return sums ? sum - counted * kBias : 0;
  }
  ZB_DEVICE u64 at_edge(int bin) const {              // the weight where a bin begins
    return power(__hiloint2double(min(bin_from + (bin << bin_shift), __double2hiint(kMiddle)), 0)) - kBias;
  }
  // The key of the smallest logit that is in a bin or above it: 5 bits of it at a time, a lane each.
  ZB_DEVICE uint32_t key_of_bin(int bin) const {
    if (bin <= 0) bin = 0;
    const int from_hi = bin_from + (bin << bin_shift);
    uint32_t lo = 0;                                 // the last one that is below
#pragma unroll 1
    for (int shift = 27; shift > -5; shift -= 5) {
      const int by = max(shift, 0);
      const uint32_t key = lo + (static_cast<uint32_t>(lane) << by);
      const bool below = key >= lo && (key < key_of(floor_x) || (key <= best && __double2hiint(log2_of(value_of(key))) < from_hi));
      lo += static_cast<uint32_t>(31 - __clz(__ballot_sync(0xffffffffu, below) | 1u)) << by;
    }
    return lo + 1;
  }
  // Where the counts (or weights) of the bins, from the highest on, reach `need`: of weights, not above *first and not below *last, by the weights at the bins' edges (one more or
  // less, for their roundings).  Returns how many logits there are from *last on; 0: the counts do not reach it.  Of counts, sh.left is what is needed of the bin.
  ZB_DEVICE uint32_t bracket(bool weights, u64 need, int* first, int* last) {
    cluster_sync();
    constexpr int kEach = (kBins + kThreads - 1) / kThreads;      // where a row has one CTA
    const int share = kBins >> (31 - __clz(ctas)), each_bins = (share + kThreads - 1) / kThreads, top_bin = kBins - 1 - rank * share - threadIdx.x * each_bins;
    uint32_t n[kEach] = {}, counted = 0;
    u64 up = 0, low = 0;
    const auto most_of = [&](int j) { return weights ? n[j] * (at_edge(top_bin - j + 1) + 1) : n[j]; };
    const auto least_of = [&](int j) { return weights ? n[j] * (max(at_edge(top_bin - j), 1ull) - 1) : n[j]; };
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (j < each_bins && static_cast<int>(threadIdx.x) * each_bins + j < share) {
#pragma unroll
        for (int c = 0; c < kMaxCtas; ++c)
          if (c < ctas) n[j] += ld_cluster_u32(zb_mapa(zb_smem_u32(&sh.hist[top_bin - j]), c));
        up += most_of(j), low += least_of(j), counted += n[j];
      }
    }
    u64 up_before = warp_upto(up, lane), low_before = warp_upto(low, lane);
    uint32_t before = counted;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    if (lane == 31) sh.part[warp] = up_before, sh.seg[warp] = low_before, sh.seg_ties[warp] = before;
    __syncthreads();
    up_before -= up, low_before -= low, before -= counted;
    up = low = 0, counted = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) up_before += sh.part[w], low_before += sh.seg[w], before += sh.seg_ties[w];
      up += sh.part[w], low += sh.seg[w], counted += sh.seg_ties[w];
    }
    if (threadIdx.x < ctas) {
      st_cluster_u64(zb_mapa(zb_smem_u32(&sh.total[rank]), threadIdx.x), up);
      st_cluster_u64(zb_mapa(zb_smem_u32(&sh.lower[rank]), threadIdx.x), low);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.ties[rank]), threadIdx.x), counted);
    }
    cluster_sync();
    up = low = 0, counted = 0;
    for (int c = 0; c < ctas; ++c) {
      if (c < rank) up_before += sh.total[c], low_before += sh.lower[c], before += sh.ties[c];
      up += sh.total[c], low += sh.lower[c], counted += sh.ties[c];
    }
    const auto tell = [&](int which, int bin, uint32_t upto, u64 left) {
      for (int c = 0; c < ctas; ++c) {
        st_cluster_u32(zb_mapa(zb_smem_u32(&sh.found[which]), c), static_cast<uint32_t>(bin));
        if (which == 0) continue;
        st_cluster_u32(zb_mapa(zb_smem_u32(&sh.found[2]), c), upto);
        st_cluster_u64(zb_mapa(zb_smem_u32(&sh.left), c), left);
      }
    };
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const u64 most = most_of(j), least = least_of(j);
      before += n[j];
      if (up_before < need && up_before + most >= need) tell(0, top_bin - j, 0, 0);
      if (low_before < need && low_before + least >= need) tell(1, top_bin - j, before, need - low_before);
      up_before += most, low_before += least;
    }
    if (rank == 0 && threadIdx.x == 0) {
      if (up < need) tell(0, 0, 0, 0);
      if (low < need) tell(1, 0, weights ? counted : 0, 0);
    }
    cluster_sync();
    *first = static_cast<int>(sh.found[0]), *last = static_cast<int>(sh.found[1]);
    return sh.found[2];
  }
  // The largest key from which on, downwards from `hi`, the counts (or weights) sum to `need`, which those from `lo` on do; *rest: what is needed there.
  // 11 bits of it at a time; over(f): f(logit) of the thread's.
  template <typename Over>
  ZB_DEVICE uint32_t narrow(bool weights, uint32_t lo, uint32_t hi, u64 need, u64* rest, Over&& over) {
    if (lo == hi) cluster_sync();                    // (as if there were a round: nobody reads what the caller's next steps write)
    while (lo != hi) {
      const int shift = max(0, 21 - __clz(hi - lo));
      for (int i = threadIdx.x; i < kBins; i += kThreads) sh.sums[i] = 0;
      __syncthreads();
      over([&](float v) {
        const uint32_t key = key_of(v);
        if (key >= lo && key <= hi) atomicAdd(&sh.sums[(key - lo) >> shift], weights ? weight(v) : 1ull);
      });
      cluster_sync();
      constexpr int kEach = (kBins + kThreads - 1) / kThreads;
      const int share = kBins >> (31 - __clz(ctas)), each_bins = (share + kThreads - 1) / kThreads, top_bin = kBins - 1 - rank * share - threadIdx.x * each_bins;
      u64 sum[kEach], before = 0, mine = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        sum[j] = 0;
        if (j < each_bins && static_cast<int>(threadIdx.x) * each_bins + j < share) {
#pragma unroll
          for (int c = 0; c < kMaxCtas; ++c)
            if (c < ctas) sum[j] += ld_cluster_u64(zb_mapa(zb_smem_u32(&sh.sums[top_bin - j]), c));
          mine += sum[j];
        }
      }
      const u64 upto = warp_upto(mine, lane);
      if (lane == 31) sh.part[warp] = upto;
      if (threadIdx.x == 0) sh.found[0] = 0, sh.left = need;      // (of a sum that does not reach it)
      __syncthreads();
      before = upto - mine, mine = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sh.part[w];
        mine += sh.part[w];
      }
      if (threadIdx.x < ctas) st_cluster_u64(zb_mapa(zb_smem_u32(&sh.total[rank]), threadIdx.x), mine);
      cluster_sync();
      for (int c = 0; c < rank; ++c) before += sh.total[c];
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (before < need && before + sum[j] >= need)
          for (int c = 0; c < ctas; ++c) {
            st_cluster_u32(zb_mapa(zb_smem_u32(&sh.found[0]), c), static_cast<uint32_t>(top_bin - j));
            st_cluster_u64(zb_mapa(zb_smem_u32(&sh.left), c), need - before);
          }
        before += sum[j];
      }
      cluster_sync();
      lo += sh.found[0] << shift;
      hi = min(hi, lo + ((1u << shift) - 1u));
      need = sh.left;
    }
    *rest = need;
    return lo;
  }
  // The key above which `need` (of counts: sh.left of the logits in the bins) is not reached; *rest: what is needed there.  The logits of the bins [last, first]
  // that are above floor_key go into the CTAs' lists, the weights of those above the bins into sh.above.
  ZB_DEVICE uint32_t cut_in(bool weights, int first, int last, uint32_t floor_key, u64 need, u64* rest) {
    const uint32_t from_key = max(key_of_bin(last), floor_key + 1);
    const float x_from = value_of(from_key), x_above = first + 1 < kBins ? value_of(max(key_of_bin(first + 1), from_key)) : INFINITY;
    const u64 left = sh.left;
    if (threadIdx.x == 0) sh.n = 0, sh.range[0] = ~0u, sh.range[1] = 0;
    __syncthreads();
    uint32_t smallest = ~0u, largest = 0, counted = 0;
    u64 above = 0;
    each([&](const float (&e)[4], int index, int step) {
      bool in[4], some = false, over = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        in[j] = e[j] >= x_from && e[j] < x_above;
        some |= in[j];
        over |= e[j] >= x_above;
      }
      if (__any_sync(0xffffffffu, over)) {           // (lanes that take no part would not be faster)
#pragma unroll
        for (int j = 0; j < 4; ++j) above += biased(e[j] >= x_above ? e[j] : -INFINITY);
        counted += 4;
      }
      if (!__any_sync(0xffffffffu, some)) return;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (in[j]) smallest = min(smallest, key_of(e[j])), largest = max(largest, key_of(e[j]));
      append(in, e, index, step);
    });
    smallest = __reduce_min_sync(0xffffffffu, smallest);
    largest = __reduce_max_sync(0xffffffffu, largest);
    above = warp_sum(above - counted * kBias);
    if (lane == 0) atomicMin(&sh.range[0], smallest), atomicMax(&sh.range[1], largest), sh.above[warp] = above;
    __syncthreads();
    if (threadIdx.x < ctas) {
      u64 a = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) a += sh.above[w];
      st_cluster_u64(zb_mapa(zb_smem_u32(&sh.total[rank]), threadIdx.x), a);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.least[rank]), threadIdx.x), sh.range[0]);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.bound[rank]), threadIdx.x), sh.range[1]);
    }
    exchange_counts();
    above = 0, listed = true;
    for (int c = 0; c < ctas; ++c) {
      smallest = min(smallest, sh.least[c]), largest = max(largest, sh.bound[c]), above += sh.total[c];
      listed = listed && sh.count[c] <= kList;
    }
    need = weights ? need - above : left;
    const int n = static_cast<int>(sh.n);
    if (listed)
      return narrow(weights, smallest, largest, need, rest, [&](auto&& f) {
        for (int i = threadIdx.x; i < n; i += kThreads) f(value_of(key_at(sh.cand[i])));
      });
    return narrow(weights, smallest, largest, need, rest, [&](auto&& f) {
      each([&](const float (&e)[4], int, int) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (e[j] == e[j]) f(e[j]);
      });
    });
  }
  // The weights of the warp's part above a cut.
  ZB_DEVICE u64 sum_above(uint32_t cut) const {
    const float cut_x = value_of(cut);
    u64 sum = 0;
    uint32_t counted = 0;
    each([&](const float (&e)[4], int, int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += biased(e[j] > cut_x ? e[j] : -INFINITY);
      counted += 4;
    });
    return warp_sum(sum - counted * kBias);
  }
  // Where the cut is among the lists: the weights of the warp's part above it, and how many equal it.
  ZB_DEVICE void sum_lists(uint32_t cut, u64* mass, uint32_t* ties) const {
    u64 m = 0;
    uint32_t t = 0;
    for (int i = lane; i < static_cast<int>(sh.n); i += 32) {
      const u64 c = sh.cand[i];
      if (index_at(c) < from || index_at(c) >= end) continue;
      if (key_at(c) > cut) m += weight(value_of(key_at(c)));
      t += key_at(c) == cut ? 1 : 0;
    }
    *mass = warp_sum(m) + sh.above[warp];
    *ties = __reduce_add_sync(0xffffffffu, t);
  }

  ZB_DEVICE void run(int row) {
    const double t = p.temperature != nullptr ? p.temperature[row] : p.temperature_all;
    const double top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p_all;
    const double min_p = p.min_p != nullptr ? p.min_p[row] : p.min_p_all;
    int top_k = p.top_k != nullptr ? p.top_k[row] : p.top_k_all;
    if (!(t > 0.0) || top_p <= 0.0) top_k = 1;
    if (top_k <= 0 || top_k > p.vocab) top_k = p.vocab;
    bool small_k = top_k > 1 && top_k <= kSmallK && top_k < p.vocab;
    // If each of n CTAs has j logits from some bound on, the row has n * j of them: the smallest of the CTAs' j-th largest is at most the row's.  CTAs at the row's end
    // that have few logits or none do not count: their j-th largest says nothing (50304 logits, of which the eighth CTA has none, with a top_k of 50: 22 us, now 11).
    const int j_th = (top_k + p.filled - 1) / p.filled;
    small_k = small_k && j_th <= kThreads;

    // ---- the row, its largest logit and its smallest one
    float most = -INFINITY, lowest = INFINITY;
    each([&](const float (&e)[4], int, int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        most = fmaxf(most, e[j]);
        lowest = e[j] > -INFINITY ? fminf(lowest, e[j]) : lowest;
      }
    });
    for (int j = threadIdx.x; j < kTable; j += kThreads) sh.table[j] = exp2((j + 0.5) / kTable);
    const uint32_t my_best = key_of(most);
    {
      const uint32_t b = __reduce_max_sync(0xffffffffu, my_best), l = __reduce_min_sync(0xffffffffu, key_of(lowest));
      if (lane == 0) sh.warp_best[warp] = b, sh.warp_least[warp] = l;
    }
    if (small_k) find_bound(my_best, j_th);
    else __syncthreads();
    zb_cluster_wait();                               // every CTA runs
    if (threadIdx.x < ctas) {
      uint32_t b = 0, l = ~0u;
      for (int w = 0; w < kWarps; ++w) b = max(b, sh.warp_best[w]), l = min(l, sh.warp_least[w]);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.best[rank]), threadIdx.x), b);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.least[rank]), threadIdx.x), l);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.bound[rank]), threadIdx.x), small_k && rank < p.filled ? sh.range[0] : ~0u);
    }
    cluster_sync();
    uint32_t row_least = ~0u, bound = ~0u;
    best = 0;
    for (int c = 0; c < ctas; ++c) best = max(best, sh.best[c]), row_least = min(row_least, sh.least[c]), bound = min(bound, sh.bound[c]);
    top = value_of(best);
    if (top == -INFINITY) {                          // nothing is allowed
      if (rank == 0 && threadIdx.x == 0) {
        p.token[row] = 0;
        if (p.logprob != nullptr) p.logprob[row] = __uint_as_float(0x7fc00000u);
      }
      return;                                        // (alike in all CTAs, and none writes to another one any more)
    }
    if (top == INFINITY) {                           // infinities are alike, and all else is nothing beside them
      kind = 1;
      top = 1.f;
      best = row_least = key_of(1.f);
      bound = min(bound, best);
    }
    // Logits, and the temperature with them, are scaled by 2^-64 where the floor below would be beyond fp32: a row whose largest is as far down as the type goes
    // (its masks' value everywhere), or one that so high a temperature makes of a few logits.  (What denormals lose of logits below 1e-19 is nothing beside such numbers.)
    double temp = t;
    if (kind == 0 && (fabsf(top) > 1e18f || (t > 1e30 && value_of(row_least) < -1e18f))) {
      kind = 2;
      temp *= 0x1p-64;
      top *= 0x1p-64f;
      best = key_of(top), row_least = key_of(value_of(row_least) * 0x1p-64f), bound = key_of(value_of(bound) * 0x1p-64f);
    }
    // Within bounds that change nothing: the next number below the largest has a weight of zero at 900 already, and logits that are not beyond 1e20 are alike at 1e36.
    // So the floor is below the largest logit and above -1e38, and -inf is not above it.
    top64 = top;
    const double next = top64 - static_cast<double>(value_of(best - (best == 0x80000000u ? 2 : 1)));      // (the key below zero's is that of no number)
    scale = fmin(t > 0.0 ? 1.4426950408889634 / fmin(temp, 1e36) : 1.0, 900.0 / next);
    floor_x = __double2float_rd(top64 - 47.0 / scale);

    // the smallest logit whose weight, rounded to 2^-53, reaches min_p
    uint32_t least = 0;
    if (min_p > 0.0) {
      const double z = log2(fmin(min_p, 1.0)) - 1.6e-16;
      const auto fits = [&](uint32_t key) { return key >= best || (static_cast<double>(value_of(key)) - top64) * scale >= z; };
      least = min(key_of(__double2float_ru(fmax(top64 + z / scale, -3.4e38))), best);
      if (!fits(least)) ++least;
      else if (fits(least - 1)) --least;
    }

    // ---- the cuts: keys above `cut` stay, and `stay` of those equal to it
    uint32_t cut = 0;
    u64 stay = ~0ull;
    if (top_k == 1) {
      cut = best;
      stay = 1;
    } else {
      if (small_k) {
        const uint32_t from_key = top_p < 1.0 ? bound : max(bound, least);      // (top_p is of the sum of all top_k)
        const int n = gather(from_key);
        if (n <= kList) {
          sort_lists(n, from_key);
          if (rank == 0) draw_from_list(row, min(n, top_k), top_p, 0, least);
          return;
        }
        cluster_sync();
      }
      const bool nucleus = top_p < 1.0;
      if (top_k < p.vocab || nucleus) {
        // Logits of no weight are never drawn.  For a nucleus alone: all logits of less than 2^z_from together are less than 1 - top_p of the sum (half of that, for
        // what sums are rounded by), which is one or more.
        const double z_from = top_k < p.vocab ? -46.0 : fmax(log2((1.0 - top_p) / (2.0 * p.vocab)) - 1e-6, -46.0);
        const bool short_list = top_k == p.vocab;
        u64 all = count_bins(z_from, row_least, nucleus, short_list);
        int first, last;
        bool done = !nucleus;
        if (nucleus) {
          __syncthreads();
          if (threadIdx.x < ctas) st_cluster_u32(zb_mapa(zb_smem_u32(&sh.count[rank]), threadIdx.x), sh.n);
          all = sum_all(all);
          if (short_list) {
            int have = 0;
            for (int c = 0; c < ctas; ++c) have += static_cast<int>(min(sh.count[c], static_cast<uint32_t>(kList + 1)));
            if (have <= kList) {
              sort_lists(have, have > 256 ? key_of_bin(0) : 0u);
              if (rank == 0) draw_from_list(row, have, top_p, all, least);
              return;
            }
          }
        }
        if (top_k < p.vocab) {
          const uint32_t n = bracket(false, top_k, &first, &last);
          if (n > 0 && n <= kList) {
            const uint32_t from_key = nucleus ? key_of_bin(last) : max(key_of_bin(last), least);
            const int have = gather(from_key);
            sort_lists(have, from_key);
            if (rank == 0) draw_from_list(row, min(have, top_k), top_p, 0, least);
            return;
          }
          if (n > 0) cut = cut_in(false, first, last, 0u, 0, &stay);
          if (n > 0 && nucleus) {
            const u64 at_cut = weight(value_of(cut));
            u64 above;
            uint32_t ties;
            if (listed) sum_lists(cut, &above, &ties);
            else above = sum_above(cut);
            cluster_sync();
            above = sum_all(lane == 0 ? above : 0);
            all = above + stay * at_cut;
            const u64 need = need_of(top_p, all);
            if (above < need) stay = (need - above + at_cut - 1) / at_cut, done = true;
            cluster_sync();
          }
        }
        if (!done) {
          const u64 need = need_of(top_p, all);
          const uint32_t n = bracket(true, need, &first, &last);
          if (n <= kList) {
            const uint32_t from_key = max(max(key_of_bin(last), cut + 1), least);
            const int have = gather(from_key);
            sort_lists(have, from_key);
            if (rank == 0) draw_from_list(row, have, top_p, all, least);
            return;
          }
          u64 rest;
          cut = cut_in(true, first, last, cut, need, &rest);
          const u64 w = weight(value_of(cut));
          stay = (rest + w - 1) / w;
        }
      }
      if (least > cut) {
        cut = least;
        stay = ~0ull;
        listed = false;
      }
    }

    // ---- what stays, CTA after CTA, warp after warp, and of the drawn one's warp eighth after eighth
    const float cut_x = value_of(cut);
    u64 mass;
    uint32_t ties;
    const auto sum_part = [&]() {                    // of the warp's part
      mass = 0, ties = 0;
      uint32_t counted = 0;
      each([&](const float (&e)[4], int, int) {
        if (cut == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) mass += biased(e[j]);
          counted += 4;
        } else if (__any_sync(0xffffffffu, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])) >= cut_x)) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mass += biased(e[j] > cut_x ? e[j] : -INFINITY);
            ties += e[j] == cut_x ? 1 : 0;
          }
          counted += 4;
        }
      });
      mass = warp_sum(mass - counted * kBias);
      ties = __reduce_add_sync(0xffffffffu, ties);
    };
    if (listed) sum_lists(cut, &mass, &ties);
    else sum_part();
    if (lane == 0) sh.seg[warp] = mass, sh.seg_ties[warp] = ties;
    __syncthreads();
    if (threadIdx.x < ctas) {
      u64 s = 0;
      uint32_t n = 0;
      for (int w = 0; w < kWarps; ++w) s += sh.seg[w], n += sh.seg_ties[w];
      st_cluster_u64(zb_mapa(zb_smem_u32(&sh.total[rank]), threadIdx.x), s);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.ties[rank]), threadIdx.x), n);
    }
    cluster_sync();
    const u64 tie_weight = cut > 0 ? weight(cut_x) : 0;
    u64 room = stay;
    const auto kept = [&](u64 m, uint32_t n) {       // of a part, whose equals of the cut stay as far as there is room
      const u64 k = min(static_cast<u64>(n), room);
      room -= k;
      return m + k * tie_weight;
    };
    u64 all = 0;
    for (int c = 0; c < ctas; ++c) all += kept(sh.total[c], sh.ties[c]);
    u64 target = target_of(uniform(row), all);
    room = stay;
    const auto pick = [&](const u64* m, const uint32_t* n, int parts) {      // the part that has the target
      for (int i = 0; i < parts; ++i) {
        const u64 before = room, here = kept(m[i], n[i]);
        if (target < here) {
          room = before;
          return i;
        }
        target -= here;
      }
      return parts - 1;                              // (there is one)
    };
    if (pick(sh.total, sh.ties, ctas) != rank) return;      // (nobody's shared memory is read from another CTA any more)
    const int owner = pick(sh.seg, sh.seg_ties, kWarps), share = p.slice / kWarps, base = rank * p.slice + owner * share, eighth = (share / kWarps + 31) / 32 * 32;
    from = min(base + warp * eighth, min(base + share, p.vocab));
    end = min(from + eighth, min(base + share, p.vocab));
    sum_part();
    if (lane == 0) sh.sub[warp] = mass, sh.sub_ties[warp] = ties;
    __syncthreads();
    if (pick(sh.sub, sh.sub_ties, kWarps) != warp) return;
    for (int i = from; i < end; i += 32) {
      const int at = i + lane;
      const float v = at < end ? fix(static_cast<float>(x[at])) : -INFINITY;
      const bool tie = cut > 0 && at < end && v == cut_x;
      const uint32_t tied = __ballot_sync(0xffffffffu, tie);
      const u64 w = tie ? (static_cast<u64>(__popc(tied & ((1u << lane) - 1u))) < room ? tie_weight : 0) : cut == 0 || v > cut_x ? weight(v) : 0;
      room -= min(room, static_cast<u64>(__popc(tied)));
      const u64 upto = warp_upto(w, lane), row_sum = __shfl_sync(0xffffffffu, upto, 31);
      if (row_sum > target) {
        if (upto > target && upto - w <= target) write(row, at, v, all);
        return;
      }
      target -= row_sum;
    }
  }
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) zb_sample_kernel(const SampleParams p, int log2_ctas) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared<kThreads>& sh = *reinterpret_cast<Shared<kThreads>*>(raw);
  zb_cluster_arrive();                               // every CTA runs before another one writes to its shared memory
  zb_pdl_launch();
  zb_pdl_wait();
  Sampler<T, kThreads> s(p, sh, log2_ctas);
  s.run(blockIdx.x >> log2_ctas);
}

template <typename T, int kThreads>
int launch(SampleParams& p, int rows, int log2, cudaStream_t s) {
  const int unit = 128 * kThreads / 32;
  p.slice = ((p.vocab + (1 << log2) - 1) / (1 << log2) + unit - 1) / unit * unit;
  p.filled = std::max(1, (p.vocab + p.slice / 4) / p.slice);
  static bool configured[16] = {};
  if (const int rc = zb_config_smem_once(zb_sample_kernel<T, kThreads>, sizeof(Shared<kThreads>), configured)) return rc;
  const cudaError_t e = zb_launch_cluster(zb_sample_kernel<T, kThreads>, dim3(static_cast<unsigned>(rows) << log2), dim3(kThreads), sizeof(Shared<kThreads>), s, 1 << log2, p, log2);
  zb_count_launch(1);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

// Eight CTAs of a row, of fewer for short ones; as many threads as the rows leave room for.
template <typename T>
int launch(SampleParams& p, int rows, cudaStream_t s) {
  int log2 = 3;
  while (log2 > 0 && (p.vocab >> log2) < 2048) --log2;
  p.vec = reinterpret_cast<uintptr_t>(p.logits) % (4 * sizeof(T)) == 0 && (rows == 1 || p.stride % 4 == 0);
  const long long ctas = static_cast<long long>(rows) << log2;
  return ctas <= 2 * zb_num_sms() ? launch<T, 512>(p, rows, log2, s) : launch<T, 256>(p, rows, log2, s);
}

}  // namespace

extern "C" {

// The arguments of a call, as the caller packs them (ops/sampling.py).
struct ZbSample {
  const void* logits;                                // [rows, vocab], fp32 or bf16, rows `stride` apart
  int32_t* token;                                    // [rows]
  float* logprob;                                    // [rows] or null
  const void* uniforms;                              // [rows] fp32 or fp64, or null
  const unsigned long long* rng;                     // {seed, draws so far} where uniforms is null
  const float *temperature, *top_p, *min_p;          // [rows] or null
  const int32_t* top_k;
  void* stream;
  long long stride;
  double temperature_all, top_p_all, min_p_all;
  int top_k_all, rows, vocab, bf16, uniforms64;
};

int zb_sample(const ZbSample* c) {
  if (c->rows <= 0) return 0;
  if (c->vocab <= 0 || c->vocab > kMaxVocab || c->rows > (1 << 24)) return -30;
  if (c->uniforms == nullptr && c->rng == nullptr) return -31;
  if (!zb_device_state()) return -20;
  SampleParams p = {};
  p.logits = c->logits;
  p.token = c->token;
  p.logprob = c->logprob;
  p.uniforms = c->uniforms;
  p.rng = c->rng;
  p.temperature = c->temperature;
  p.top_p = c->top_p;
  p.min_p = c->min_p;
  p.top_k = c->top_k;
  p.stride = c->stride;
  p.temperature_all = c->temperature_all;
  p.top_p_all = c->top_p_all;
  p.min_p_all = c->min_p_all;
  p.top_k_all = c->top_k_all;
  p.vocab = c->vocab;
  p.uniforms64 = c->uniforms64;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(c->stream);
  return c->bf16 ? launch<__nv_bfloat16>(p, c->rows, s) : launch<float>(p, c->rows, s);
}

}  // extern "C"
