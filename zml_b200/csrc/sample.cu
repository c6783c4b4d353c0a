// The draw of one token for each row of logits, with temperature, top-k, top-p and min-p of every row, from given random numbers.
//
// With M = max x, w_i = 2^((x_i - M) log2(e) / T): the top_k largest stay (equal ones: the lower indices); of these, in the order of their size, those
// whose predecessors' weights are less than top_p of the sum; of these, those with w_i >= min_p.  The token is the first in the vocabulary's order up to which the
// weights that stayed sum to more than u times their sum.
//
// Weights are whole numbers of 2^-44.  Sums of up to 2^18 of them are exact in 64 bits and do not depend on an order; a sum is off by at most 2^-27 and
// typically 2^-36 of the largest weight.  (A sum of fp32 weights is off by 1e-7 of the whole, and among 128 thousand flat weights each is 8e-6 of it:
// one draw in a hundred would be another token.)
//
// A cluster of CTAs holds a row in shared memory, a slice a CTA, and reads it from there as often as it needs; the row is not sorted.  All cuts keep
// what is in front in the order of size, so a row ends in one of two ways:
//   * a list: what is at least as large as a bound that is known beforehand (the k-th largest of some logits; the weight below which all of the vocabulary
//     together is less than 1 - top_p; min_p) is usually a few hundred logits, which one CTA ranks, sums and draws from;
//   * a cut: where these are too many, a histogram finds the smallest logit that stays and how many of its equals do, every warp sums the weights
//     of its part, and the warp that has the drawn one looks for it.
// What bounds it: the logits' bytes for many rows, beside some 30 instructions of a weight where the whole row's sum is needed; for few rows the passes' and
// the cluster's barriers' latency.
#include "common.cuh"
#include "host_api.h"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCtas = 8;
constexpr int kMaxSlice = 49152;                     // logits of a CTA
constexpr int kList = 1024;
constexpr int kSmallK = 256;
constexpr int kBins = 2048;
constexpr int kTable = 512;                          // 2^((j + 1/2) / 512)
constexpr double kOne = 17592186044416.0;            // 2^44
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
  int top_k_all, vocab, slice, uniforms64, vec;  // vec: every row starts on four logits
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

struct Shared {
  double table[kTable];
  union {
    struct {
      u64 cand[kList];                               // of this CTA: key << 32 | ~index, the larger, the further in front
      u64 sorted[kList];                             // CTA 0: of the cluster
      u64 weight[kList];
    } list;
    uint32_t hist[3][kBins];                         // counts, or 15 bits each of the weights
  };
  u64 part[2][kWarps];
  u64 total[kMaxCtas];                               // of every CTA
  uint32_t ties[kMaxCtas], count[kMaxCtas], best[kMaxCtas], bound[kMaxCtas], least[kMaxCtas];
  uint32_t warp_ties[kWarps], warp_best[kWarps], warp_least[kWarps], top[kWarps * (kSmallK / kWarps + 1)], n, range[2];
  u64 left;                                          // what CTA 0 has found, in every CTA
  uint32_t found;
};

// All threads of a cluster, which is one row.
template <typename T>
struct Sampler {
  const SampleParams& p;
  Shared& sh;
  float* x_s;                    // the CTA's slice
  int ctas, rank, warp, lane, from, rows, first;      // a warp has `rows` rows of 128 logits of the slice, from `first` on, four neighbours a lane
  float top, floor_x;            // the largest logit; below floor_x weights are zero
  double top64, scale;           // log2 of a weight is (x - top) * scale
  uint32_t best;

  ZB_DEVICE Sampler(const SampleParams& params, Shared& shared, float* x, int log2_ctas)
      : p(params), sh(shared), x_s(x), ctas(1 << log2_ctas), rank(blockIdx.x & (ctas - 1)), warp(threadIdx.x >> 5), lane(threadIdx.x & 31) {
    from = rank * p.slice;
    rows = p.slice / (128 * kWarps);
    first = warp * rows * 128;
  }

  // The weight of a logit that is not above `top`, in 2^-44, plus kBias.  z is held with 41 bits behind the point: 9 of them choose the table's entry, with the
  // other 32 as r, around their middle, 2^r is a cubic (off by 9e-15).
  ZB_DEVICE u64 biased(float x) const {
    const double t = __fma_rn(static_cast<double>(fmaxf(x, floor_x)) - top64, scale, 3072.0);
    const int hi = __double2hiint(t);
    const double r = __hiloint2double(0x43300000, __double2loint(t)) - 4503601774854144.0;      // 2^52 + 2^31
    constexpr double c1 = 0.6931471805599453 * 0x1p-41, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
    const double base = sh.table[hi & (kTable - 1)];
    const double b = __hiloint2double(__double2hiint(base) + ((hi & ~(kTable - 1)) << 11) - (1024 << 20), __double2loint(base));
    const double q = __fma_rn(__fma_rn(r, c3, c2), r, c1) * r;
    return static_cast<u64>(__double_as_longlong(__fma_rn(b, q, b) + 256.0));
  }
  ZB_DEVICE u64 weight(float x) const { return biased(x) - kBias; }

  template <typename F>
  ZB_DEVICE void each(F&& f) const {                 // f(index in the slice of the first, four logits): the warp's, in order
#pragma unroll 1
    for (int i = 0; i < rows; ++i) {
      const int at = first + i * 128 + lane * 4;
      f(at, *reinterpret_cast<const float4*>(x_s + at));
    }
  }

  ZB_DEVICE void load(const T* x, float& most, float& least) {
    const auto take = [&](float v) {
      v = v != v ? -INFINITY : v;
      most = fmaxf(most, v);
      least = v > -INFINITY ? fminf(least, v) : least;
      return v;
    };
    most = -INFINITY, least = INFINITY;
    const int whole = min(rows, max(0, (p.vocab - from - first) / 128));      // rows without an end
    int i = 0;
    if (p.vec) {
#pragma unroll 4
      for (; i < whole; ++i) {
        const int at = first + i * 128 + lane * 4;
        float4 v;
        if constexpr (sizeof(T) == 4) {
          v = *reinterpret_cast<const float4*>(x + from + at);
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(x + from + at);
          v = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
        }
        *reinterpret_cast<float4*>(x_s + at) = make_float4(take(v.x), take(v.y), take(v.z), take(v.w));
      }
    }
#pragma unroll 2
    for (; i < rows; ++i) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = from + first + i * 128 + j * 32 + lane;
        v[j] = at < p.vocab ? static_cast<float>(x[at]) : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) x_s[first + i * 128 + j * 32 + lane] = take(v[j]);
    }
    __syncwarp();
  }

  // The k-th largest of at least k of the CTA's logits: each warp's largest few of its lanes' largest.
  ZB_DEVICE void find_bound(uint32_t mine, int k) {
    const int per_warp = min((k + kWarps - 1) / kWarps + 1, 32);
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
      for (int j = 0; j < kWarps * per_warp; ++j) ahead += sh.top[j] > m || (sh.top[j] == m && j < static_cast<int>(threadIdx.x)) ? 1 : 0;
      if (ahead == k - 1) sh.range[0] = m;
    }
    __syncthreads();
  }

  // Over the cluster, in every thread; *before: of the CTAs in front, *front: and of the warps in front.
  ZB_DEVICE u64 sum_all(u64 v) {
    v = warp_sum(v);
    if (lane == 0) sh.part[0][warp] = v;
    __syncthreads();
    if (warp == 0) {
      u64 s = lane < kWarps ? sh.part[0][lane] : 0;
      s = warp_sum(s);
      if (lane < ctas) st_cluster_u64(zb_mapa(zb_smem_u32(&sh.total[rank]), lane), s);
    }
    cluster_sync();
    u64 s = 0;
    for (int c = 0; c < ctas; ++c) s += sh.total[c];
    return s;
  }

  // A row's logits from key `lo` on into the CTAs' lists; how many in the cluster.  (Another barrier has to come before the lists are written again.)
  ZB_DEVICE int gather(uint32_t lo) {
    const float bound = value_of(lo);
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    each([&](int at, const float4& v) {
      if (!__any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= bound)) return;
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e[j] >= bound && from + at + j < p.vocab) {
          const uint32_t slot = atomicAdd(&sh.n, 1u);
          if (slot < kList) sh.list.cand[slot] = static_cast<u64>(key_of(e[j])) << 32 | static_cast<uint32_t>(~(from + at + j));
        }
    });
    __syncthreads();
    if (threadIdx.x < ctas) st_cluster_u32(zb_mapa(zb_smem_u32(&sh.count[rank]), threadIdx.x), sh.n);
    cluster_sync();
    int n = 0;
    for (int c = 0; c < ctas; ++c) n += static_cast<int>(min(sh.count[c], static_cast<uint32_t>(kList + 1)));
    return n;
  }

  // The CTAs' lists, n in all, to CTA 0, in the order of size.
  ZB_DEVICE void sort_lists(int n) {
    if (rank == 0) {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        int c = 0, at = i;
        while (at >= static_cast<int>(sh.count[c])) at -= sh.count[c++];
        sh.list.weight[i] = ld_cluster_u64(zb_mapa(zb_smem_u32(&sh.list.cand[at]), c));
      }
    }
    cluster_sync();                                  // nobody leaves or writes its list before it has been read
    if (rank != 0) return;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const u64 mine = sh.list.weight[i];
      int ahead = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) ahead += sh.list.weight[j] > mine ? 1 : 0;
      sh.list.sorted[ahead] = mine;
    }
    __syncthreads();
  }
  static ZB_DEVICE uint32_t key_at(u64 c) { return static_cast<uint32_t>(c >> 32); }
  static ZB_DEVICE int index_at(u64 c) { return ~static_cast<int>(static_cast<uint32_t>(c)); }

  // Sums up to each of the first n of the sorted list (CTA 0): of two neighbours a thread, those in front of the first.
  ZB_DEVICE u64 list_before(int n, u64& w0, u64& w1, u64& all) {
    const int i = 2 * threadIdx.x;
    w0 = i < n ? weight(value_of(key_at(sh.list.sorted[i]))) : 0;
    w1 = i + 1 < n ? weight(value_of(key_at(sh.list.sorted[i + 1]))) : 0;
    const u64 upto = warp_upto(w0 + w1, lane);
    if (lane == 31) sh.part[0][warp] = upto;
    __syncthreads();
    u64 before = upto - w0 - w1;
    all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.part[0][w];
      all += sh.part[0][w];
    }
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
    u64 w0, w1, sum;
    u64 before = list_before(n, w0, w1, sum);
    const int i = 2 * threadIdx.x;
    const u64 need = top_p < 1.0 ? need_of(top_p, all != 0 ? all : sum) : ~0ull;
    const bool s0 = i < n && (i == 0 || (before < need && key_at(sh.list.sorted[i]) >= least));
    const bool s1 = i + 1 < n && before + w0 < need && key_at(sh.list.sorted[i + 1]) >= least;
    if (i < n) sh.list.weight[i] = w0;
    if (i + 1 < n) sh.list.weight[i + 1] = w1;
    const int m = __syncthreads_count(s0) + __syncthreads_count(s1);      // those in front stay
    // their sum
    if ((s0 && i == m - 1) || (s1 && i + 1 == m - 1)) sh.left = before + w0 + (s1 ? w1 : 0);
    __syncthreads();
    const u64 kept = sh.left, target = target_of(uniform(row), kept);
    for (int a = threadIdx.x; a < m; a += kThreads) {
      const u64 mine = sh.list.sorted[a];
      const uint32_t idx = static_cast<uint32_t>(mine);      // complements: larger is further in front
      u64 s = 0;
#pragma unroll 4
      for (int j = 0; j < m; ++j) s += static_cast<uint32_t>(sh.list.sorted[j]) > idx ? sh.list.weight[j] : 0;
      if (s <= target && target - s < sh.list.weight[a]) write(row, index_at(mine), value_of(key_at(mine)), kept);
    }
  }

  // The largest key up to which, from above, the counts (or weights) of the logits above `floor_key` sum to at least `need`; *rest: what is needed there.
  // A histogram over 2048 equal intervals of [value_of(lo), top], and a list of the interval that has it - or, where that is too long, what its keys have in
  // common is looked for bit by bit.
  template <bool WEIGHTS>
  ZB_DEVICE uint32_t search(uint32_t lo, uint32_t floor_key, u64 need, u64* rest) {
    const float x_lo = fmaxf(value_of(lo), -3.0e38f), span = top - x_lo, by = span > 0.f ? static_cast<float>(kBins - 1) / span : 0.f;
    const auto bin_of = [&](float x) { return max(0, min(kBins - 1, static_cast<int>((x - x_lo) * by))); };      // grows with x
    for (int i = threadIdx.x; i < 3 * kBins; i += kThreads) (&sh.hist[0][0])[i] = 0;
    __syncthreads();
    each([&](int, const float4& v) {
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!(e[j] >= x_lo) || key_of(e[j]) <= floor_key) continue;
        const int b = bin_of(e[j]);
        if (WEIGHTS) {
          const u64 w = weight(e[j]);
          atomicAdd(&sh.hist[0][b], static_cast<uint32_t>(w) & 0x7fffu);
          atomicAdd(&sh.hist[1][b], static_cast<uint32_t>(w >> 15) & 0x7fffu);
          atomicAdd(&sh.hist[2][b], static_cast<uint32_t>(w >> 30));
        } else {
          atomicAdd(&sh.hist[0][b], 1u);
        }
      }
    });
    cluster_sync();
    if (rank == 0) {
      // sums of four bins a thread, from the highest on
      const int bin0 = kBins - 4 - 4 * threadIdx.x;
      u64 b[4] = {0, 0, 0, 0};
      for (int c = 0; c < ctas; ++c)
#pragma unroll
        for (int k = 0; k < (WEIGHTS ? 3 : 1); ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] += static_cast<u64>(ld_cluster_u32(zb_mapa(zb_smem_u32(&sh.hist[k][bin0 + j]), c))) << (15 * k);
      const u64 sum = b[0] + b[1] + b[2] + b[3], upto = warp_upto(sum, lane);
      if (lane == 31) sh.part[0][warp] = upto;
      __syncthreads();
      u64 before = upto - sum;
      for (int w = 0; w < warp; ++w) before += sh.part[0][w];
      if (before < need && before + sum >= need) {
        int j = 3;
        while (j > 0 && before + b[j] < need) before += b[j--];
        for (int c = 0; c < ctas; ++c) {
          st_cluster_u64(zb_mapa(zb_smem_u32(&sh.left), c), need - before);
          st_cluster_u32(zb_mapa(zb_smem_u32(&sh.found), c), static_cast<uint32_t>(bin0 + j));
        }
      }
      if (threadIdx.x == kThreads - 1 && before + sum < need)      // there are not as many
        for (int c = 0; c < ctas; ++c) st_cluster_u32(zb_mapa(zb_smem_u32(&sh.found), c), ~0u);
    }
    cluster_sync();
    const int bin = static_cast<int>(sh.found);
    need = sh.left;
    if (bin < 0) {
      *rest = ~0ull;
      cluster_sync();
      return 0;
    }
    const auto inside = [&](float x) { return x >= x_lo && key_of(x) > floor_key && bin_of(x) == bin; };
    // ---- the interval's logits
    if (threadIdx.x == 0) sh.n = 0, sh.range[0] = ~0u, sh.range[1] = 0;
    __syncthreads();
    uint32_t smallest = ~0u, largest = 0;
    each([&](int at, const float4& v) {
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!inside(e[j])) continue;
        const uint32_t key = key_of(e[j]), slot = atomicAdd(&sh.n, 1u);
        smallest = min(smallest, key), largest = max(largest, key);
        if (slot < kList) sh.list.cand[slot] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~(from + at + j));
      }
    });
    smallest = __reduce_min_sync(0xffffffffu, smallest);
    largest = __reduce_max_sync(0xffffffffu, largest);
    if (lane == 0) atomicMin(&sh.range[0], smallest), atomicMax(&sh.range[1], largest);
    __syncthreads();
    if (threadIdx.x < ctas) {
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.count[rank]), threadIdx.x), sh.n);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.least[rank]), threadIdx.x), sh.range[0]);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.bound[rank]), threadIdx.x), sh.range[1]);
    }
    cluster_sync();
    int n = 0;
    for (int c = 0; c < ctas; ++c) {
      n += static_cast<int>(min(sh.count[c], static_cast<uint32_t>(kList + 1)));
      smallest = min(smallest, sh.least[c]), largest = max(largest, sh.bound[c]);
    }
    if (smallest == largest) {
      *rest = need;
      cluster_sync();
      return smallest;
    }
    if (n <= kList) {
      sort_lists(n);
      if (rank == 0) {
        u64 w0, w1, all;
        u64 before;
        const int i = 2 * threadIdx.x;
        if (WEIGHTS) {
          before = list_before(n, w0, w1, all);
        } else {
          before = i;
          w0 = i < n, w1 = i + 1 < n;
        }
        // the first whose sum reaches it; what its equals in front of it have is part of `rest`
        const bool here0 = i < n && before < need && before + w0 >= need, here1 = i + 1 < n && before + w0 < need && before + w0 + w1 >= need;
        if (here0 || here1) {
          const int at = here0 ? i : i + 1;
          const uint32_t key = key_at(sh.list.sorted[at]);
          u64 left = need - (here0 ? before : before + w0);
          const u64 w = WEIGHTS ? weight(value_of(key)) : 1;
          for (int j = at - 1; j >= 0 && key_at(sh.list.sorted[j]) == key; --j) left += w;
          for (int c = 0; c < ctas; ++c) {
            st_cluster_u64(zb_mapa(zb_smem_u32(&sh.left), c), left);
            st_cluster_u32(zb_mapa(zb_smem_u32(&sh.found), c), key);
          }
        }
      }
      cluster_sync();
      *rest = sh.left;
      const uint32_t key = sh.found;
      cluster_sync();
      return key;
    }
    // ---- bit by bit, from the highest one in which they differ: whether what has it set is enough
    uint32_t prefix = smallest;
    for (int bit = 31 - __clz(smallest ^ largest); bit >= 0; --bit) {
      const uint32_t mask = ~((1u << bit) - 1u), want = (prefix & (mask << 1)) | 1u << bit;
      u64 sum = 0;
      each([&](int, const float4& v) {
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (inside(e[j]) && (key_of(e[j]) & mask) == want) sum += WEIGHTS ? weight(e[j]) : 1;
      });
      cluster_sync();
      sum = sum_all(sum);
      if (sum >= need) {
        prefix = want;
      } else {
        need -= sum;
        prefix = want & ~(1u << bit);
      }
    }
    cluster_sync();
    *rest = need;
    return prefix;
  }

  ZB_DEVICE void run(int row) {
    const T* x = reinterpret_cast<const T*>(p.logits) + static_cast<size_t>(row) * p.stride;
    const double t = p.temperature != nullptr ? p.temperature[row] : p.temperature_all;
    const double top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p_all;
    const double min_p = p.min_p != nullptr ? p.min_p[row] : p.min_p_all;
    int top_k = p.top_k != nullptr ? p.top_k[row] : p.top_k_all;
    if (!(t > 0.0) || top_p <= 0.0) top_k = 1;
    if (top_k <= 0 || top_k > p.vocab) top_k = p.vocab;
    bool small_k = top_k > 1 && top_k <= kSmallK && top_k < p.vocab;

    // ---- the row, its largest logit and its smallest one
    float most, lowest;
    load(x, most, lowest);
    for (int j = threadIdx.x; j < kTable; j += kThreads) sh.table[j] = exp2((j + 0.5) / kTable);
    const uint32_t my_best = key_of(most);
    {
      const uint32_t b = __reduce_max_sync(0xffffffffu, my_best), l = __reduce_min_sync(0xffffffffu, key_of(lowest));
      if (lane == 0) sh.warp_best[warp] = b, sh.warp_least[warp] = l;
    }
    if (small_k) find_bound(my_best, top_k);
    else __syncthreads();
    zb_cluster_wait();                               // every CTA runs
    if (threadIdx.x < ctas) {
      uint32_t b = 0, l = ~0u;
      for (int w = 0; w < kWarps; ++w) b = max(b, sh.warp_best[w]), l = min(l, sh.warp_least[w]);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.best[rank]), threadIdx.x), b);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.least[rank]), threadIdx.x), l);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.bound[rank]), threadIdx.x), small_k ? sh.range[0] : 0u);
    }
    cluster_sync();
    uint32_t row_least = ~0u, bound = 0;
    best = 0;
    for (int c = 0; c < ctas; ++c) best = max(best, sh.best[c]), row_least = min(row_least, sh.least[c]), bound = max(bound, sh.bound[c]);
    top = value_of(best);
    if (top == -INFINITY) {                          // nothing is allowed
      if (rank == 0 && threadIdx.x == 0) {
        p.token[row] = 0;
        if (p.logprob != nullptr) p.logprob[row] = __uint_as_float(0x7fc00000u);
      }
      return;                                        // (alike in all CTAs, and none writes to another one any more)
    }
    if (top == INFINITY) {                           // infinities are alike, and all else is nothing beside them
      each([&](int at, const float4& v) {
        *reinterpret_cast<float4*>(x_s + at) = make_float4(v.x == INFINITY ? 1.f : -INFINITY, v.y == INFINITY ? 1.f : -INFINITY, v.z == INFINITY ? 1.f : -INFINITY, v.w == INFINITY ? 1.f : -INFINITY);
      });
      __syncwarp();
      top = 1.f;
      best = row_least = key_of(1.f);
      bound = min(bound, best);
    }
    if (t > 1e37 && (top > 1e30f || value_of(row_least) < -1e30f)) {      // so that the scale below leaves them alike
      each([&](int at, const float4& v) {
        *reinterpret_cast<float4*>(x_s + at) = make_float4(v.x * 0x1p-100f, v.y * 0x1p-100f, v.z * 0x1p-100f, v.w * 0x1p-100f);
      });
      __syncwarp();
      top *= 0x1p-100f;
      best = key_of(top), row_least = key_of(value_of(row_least) * 0x1p-100f), bound = key_of(value_of(bound) * 0x1p-100f);
    }
    // Within bounds that change nothing: the next number below the largest has a weight of zero at 900 already, and at 1e37 all finite ones are alike.
    top64 = top;
    const double next = best > 0x00800000u ? top64 - static_cast<double>(value_of(best - 1)) : 1.0;
    scale = t > 0.0 ? fmin(1.4426950408889634 / fmin(t, 1e37), 900.0 / next) : 1.0;
    floor_x = __double2float_rd(fmax(top64 - 47.0 / scale, -3.4e38));

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
        const int n = gather(max(bound, least));
        if (n <= kList) {
          sort_lists(n);
          if (rank == 0) draw_from_list(row, min(n, top_k), top_p, 0, least);
          return;
        }
        cluster_sync();
      }
      if (top_k < p.vocab) cut = search<false>(row_least, 0u, top_k, &stay);
      u64 all = 0;
      if (top_p < 1.0) {
        u64 above = 0;
        uint32_t n = 0;
        each([&](int, const float4& v) {
          const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const u64 w = biased(e[j]);
            if (cut == 0 || key_of(e[j]) > cut) above += w, ++n;
          }
        });
        above = sum_all(above - n * kBias);
        cluster_sync();
        const u64 at_cut = cut > 0 ? weight(value_of(cut)) : 0;
        all = above + (cut > 0 ? stay * at_cut : 0);
        // All logits below this weight together are less than 1 - top_p of the sum (half of that, for what sums are rounded by)
        const double z = log2(static_cast<double>(all) / kOne * (1.0 - top_p) / (2.0 * p.vocab)) - 1e-6;
        const uint32_t enough = max(key_of(__double2float_rd(fmax(top64 + z / scale, -3.4e38))), 1u);
        const u64 need = need_of(top_p, all);
        if (enough > cut) {
          const int n = gather(max(enough, least));
          if (n <= kList) {
            sort_lists(n);
            if (rank == 0) draw_from_list(row, n, top_p, all, least);
            return;
          }
          cluster_sync();
        }
        if (above >= need) {
          u64 rest;
          const uint32_t old = cut;
          cut = search<true>(max(enough, row_least), old, need, &rest);
          const u64 w = weight(value_of(cut));
          stay = (rest + w - 1) / w;
        } else {
          stay = (need - above + at_cut - 1) / at_cut;
        }
      } else if (least > cut) {
        const int n = gather(least);
        if (n <= kList) {
          sort_lists(n);
          if (rank == 0) draw_from_list(row, n, 2.0, 0, least);
          return;
        }
        cluster_sync();
      }
      if (least > cut) {
        cut = least;
        stay = ~0ull;
      }
    }

    // ---- what stays, warp after warp and CTA after CTA
    u64 mass = 0;
    uint32_t ties = 0, counted = 0;
    const float cut_x = value_of(cut);
    each([&](int, const float4& v) {
      const float e[4] = {v.x, v.y, v.z, v.w};
      if (cut == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) mass += biased(e[j]);
        counted += 4;
      } else if (__any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= cut_x)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (e[j] > cut_x) mass += biased(e[j]), ++counted;
          ties += e[j] == cut_x ? 1 : 0;
        }
      }
    });
    mass = warp_sum(mass - counted * kBias);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) sh.part[1][warp] = mass, sh.warp_ties[warp] = ties;
    __syncthreads();
    if (threadIdx.x < ctas) {
      u64 s = 0;
      uint32_t n = 0;
      for (int w = 0; w < kWarps; ++w) s += sh.part[1][w], n += sh.warp_ties[w];
      st_cluster_u64(zb_mapa(zb_smem_u32(&sh.total[rank]), threadIdx.x), s);
      st_cluster_u32(zb_mapa(zb_smem_u32(&sh.ties[rank]), threadIdx.x), n);
    }
    cluster_sync();
    const u64 tie_weight = cut > 0 ? weight(cut_x) : 0;
    const auto kept = [&](u64 m, uint32_t n, u64& room) {      // of a part, whose equals of the cut stay as far as there is room
      const u64 k = min(static_cast<u64>(n), room);
      room -= k;
      return m + k * tie_weight;
    };
    u64 all = 0, room = stay;
    for (int c = 0; c < ctas; ++c) all += kept(sh.total[c], sh.ties[c], room);
    u64 target = target_of(uniform(row), all);
    room = stay;
    for (int c = 0; c < ctas; ++c) {
      const u64 before = room, here = kept(sh.total[c], sh.ties[c], room);
      if (target >= here) {
        target -= here;
        continue;
      }
      if (c != rank) return;                         // (nobody's shared memory is read from another CTA any more)
      room = before;
      break;
    }
    for (int w = 0; w < kWarps; ++w) {
      const u64 before = room, here = kept(sh.part[1][w], sh.warp_ties[w], room);
      if (target >= here) {
        target -= here;
        continue;
      }
      if (w != warp) return;
      room = before;
      break;
    }
#pragma unroll 1
    for (int i = 0; i < rows; ++i) {
      const int at = first + i * 128 + lane * 4;
      const float4 v = *reinterpret_cast<const float4*>(x_s + at);
      const float e[4] = {v.x, v.y, v.z, v.w};
      uint32_t mine = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) mine += cut > 0 && e[j] == cut_x ? 1 : 0;
      uint32_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
      }
      u64 tie = upto - mine, w[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = cut == 0 || e[j] > cut_x ? weight(e[j]) : 0;
        if (cut > 0 && e[j] == cut_x && tie++ < room) w[j] = tie_weight;
        sum += w[j];
      }
      room -= min(room, static_cast<u64>(__shfl_sync(0xffffffffu, upto, 31)));
      const u64 sums = warp_upto(sum, lane), row_sum = __shfl_sync(0xffffffffu, sums, 31);
      if (row_sum > target) {
        u64 s = sums - sum;
        if (s <= target && sums > target) {
          int j = 0;
          while (s + w[j] <= target) s += w[j++];
          write(row, from + at + j, e[j], all);
        }
        return;
      }
      target -= row_sum;
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) zb_sample_kernel(const SampleParams p, int log2_ctas) {
  extern __shared__ __align__(16) float x_s[];       // [slice]
  __shared__ Shared sh;
  zb_cluster_arrive();                               // every CTA runs before another one writes to its shared memory
  zb_pdl_launch();
  zb_pdl_wait();
  Sampler<T> s(p, sh, x_s, log2_ctas);
  s.run(blockIdx.x >> log2_ctas);
}

// CTAs of a row: as many as keep its slices small enough for two on an SM, and more while that fills the GPU.
int ctas_of(int rows, int vocab, int sms) {
  int log2 = 0;
  while (log2 < 3 && ((vocab + (1 << log2) - 1) >> log2) > 20480) ++log2;
  while (log2 < 3 && (static_cast<long long>(rows) << log2) < 2 * sms && (vocab >> log2) > 4 * kThreads) ++log2;
  return log2;
}

template <typename T>
int launch(SampleParams& p, int rows, cudaStream_t s) {
  const int log2 = ctas_of(rows, p.vocab, zb_num_sms()), unit = 128 * kWarps;
  p.slice = ((p.vocab + (1 << log2) - 1) / (1 << log2) + unit - 1) / unit * unit;
  p.vec = reinterpret_cast<uintptr_t>(p.logits) % (4 * sizeof(T)) == 0 && (rows == 1 || p.stride % 4 == 0);
  static bool configured[16] = {};
  if (const int rc = zb_config_smem_once(zb_sample_kernel<T>, kMaxSlice * 4, configured)) return rc;
  const cudaError_t e = zb_launch_cluster(zb_sample_kernel<T>, dim3(static_cast<unsigned>(rows) << log2), dim3(kThreads), p.slice * 4, s, 1 << log2, p, log2);
  zb_count_launch(1);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
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
  if (c->vocab <= 0 || c->vocab > kMaxSlice * kMaxCtas || c->rows > (1 << 24)) return -30;
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
