// The draw of one token for each row of logits, with temperature, top-k, top-p and min-p of every row, from given random numbers.
//
// With M = max x, w_i = 2^((x_i - M) log2(e) / T): the top_k largest stay (equal ones: the lower indices); of these, in the order of their size, those
// whose predecessors' weights are less than top_p of the sum; of these, those with w_i >= min_p.  The token is the first in the vocabulary's order up to which the
// weights that stayed sum to more than u times their sum.
//
// All three cuts end in the same form: a key (the order-preserving integer image of a logit) and how many of the logits equal to it stay, the first
// ones.  So the row is not sorted.
//
// Weights are whole numbers of 2^-44.  Sums of up to 2^18 of them are exact in 64 bits and do not depend on an order; a sum is off by at most 2^-27 and
// typically 2^-36 of the largest weight.  (A sum of fp32 weights is off by 1e-7 of the whole, and among 128 thousand flat weights each is 8e-6 of it:
// one draw in a hundred would be another token.)
//
// A cluster of CTAs holds a row in shared memory and reads it from there as often as it needs.
#include "common.cuh"
#include "host_api.h"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCtas = 8;
constexpr int kMaxSlice = 49152;                     // logits of a CTA
constexpr int kBits = 11, kBins = 1 << kBits;
constexpr double kOne = 17592186044416.0;            // 2^44

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
  int top_k_all, vocab, slice, uniforms64;
};

// Order-preserving; one zero.  NaN does not come here.
ZB_DEVICE uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
ZB_DEVICE float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

ZB_DEVICE double uniform53(unsigned long long seed, unsigned long long draw, int row) {
  // splitmix64 of (seed, draw, row)
  uint64_t z = seed + 0x9e3779b97f4a7c15ull * (draw * 0x100000000ull + static_cast<uint64_t>(row) + 1);
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  z ^= z >> 31;
  return static_cast<double>(z >> 11) * 0x1p-53;
}

ZB_DEVICE void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
ZB_DEVICE void st_cluster_u64(uint32_t addr, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
ZB_DEVICE unsigned long long ld_cluster_u64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

struct Shared {
  unsigned long long hist[kBins];
  unsigned long long part[kThreads];
  unsigned long long mass[kMaxCtas * kWarps];        // CTA 0: every warp's
  uint32_t ties[kMaxCtas * kWarps];
  uint32_t most[kMaxCtas];
  // what CTA 0 has found, in every CTA
  unsigned long long left;                           // of what is looked for, at the keys not yet decided
  unsigned long long target;
  uint32_t prefix, pad;
  int owner;
};

ZB_DEVICE void cluster_sync() {
  zb_cluster_arrive();
  zb_cluster_wait();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) zb_sample_kernel(const SampleParams p, int log2_ctas) {
  extern __shared__ __align__(16) float x_s[];       // [slice]
  __shared__ Shared sh;
  const int ctas = 1 << log2_ctas, rank = blockIdx.x & (ctas - 1), row = blockIdx.x >> log2_ctas, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  zb_cluster_arrive();                               // every CTA runs before another one writes to its shared memory
  zb_pdl_launch();
  zb_pdl_wait();
  const T* x = reinterpret_cast<const T*>(p.logits) + static_cast<size_t>(row) * p.stride;
  const int from = rank * p.slice;
  // A warp has a part of the slice, in rows of 128 logits, four neighbours a lane.
  const int rows_of_warp = p.slice / 128 / kWarps, first = warp * rows_of_warp * 128;
  const double t = p.temperature != nullptr ? p.temperature[row] : p.temperature_all;
  const double top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p_all;
  const double min_p = p.min_p != nullptr ? p.min_p[row] : p.min_p_all;
  int top_k = p.top_k != nullptr ? p.top_k[row] : p.top_k_all;
  if (!(t > 0.0) || top_p <= 0.0) top_k = 1;
  if (top_k <= 0 || top_k > p.vocab) top_k = p.vocab;

  // ---- the row, and its largest logit
  float most = -INFINITY;
  for (int i = 0; i < rows_of_warp; ++i) {
    float4 v;
    float* e = reinterpret_cast<float*>(&v);
    const int at = first + i * 128 + lane * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int idx = from + at + j;
      e[j] = idx < p.vocab ? static_cast<float>(x[idx]) : -INFINITY;
      if (isnan(e[j])) e[j] = -INFINITY;
      most = fmaxf(most, e[j]);
    }
    *reinterpret_cast<float4*>(x_s + at) = v;
  }
  sh.part[threadIdx.x] = 0;
  const uint32_t warp_most = __reduce_max_sync(0xffffffffu, key_of(most));
  __shared__ uint32_t warp_key[kWarps];
  if (lane == 0) warp_key[warp] = warp_most;
  __syncthreads();
  zb_cluster_wait();
  if (threadIdx.x < ctas) {
    uint32_t m = 0;
    for (int w = 0; w < kWarps; ++w) m = max(m, warp_key[w]);
    st_cluster_u32(zb_mapa(zb_smem_u32(&sh.most[rank]), threadIdx.x), m);
  }
  cluster_sync();
  uint32_t best = 0;
  for (int c = 0; c < ctas; ++c) best = max(best, sh.most[c]);
  const float top = value_of(best);
  if (top == -INFINITY) {                            // nothing is allowed
    if (rank == 0 && threadIdx.x == 0) {
      p.token[row] = 0;
      if (p.logprob != nullptr) p.logprob[row] = __uint_as_float(0x7fc00000u);
    }
    return;                                          // (alike in all CTAs, and none has written to another since the barrier)
  }
  const double scale = t > 0.0 ? 1.4426950408889634 / t : 1.0, top64 = top;
  const auto weight = [&](float v) -> unsigned long long {
    if (v == top) return 1ull << 44;
    const double z = (static_cast<double>(v) - top64) * scale;
    return z >= -46.0 ? __double2ull_rn(exp2(z) * kOne) : 0ull;
  };
  const auto each = [&](auto&& f) {                  // the warp's logits in order, four a lane
    for (int i = 0; i < rows_of_warp; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(x_s + first + i * 128 + lane * 4);
      f(i, v);
    }
  };
  const auto block_sum = [&](unsigned long long v) { // over the cluster, in every thread
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane < ctas) st_cluster_u64(zb_mapa(zb_smem_u32(&sh.mass[rank * kWarps + warp]), lane), v);
    cluster_sync();
    unsigned long long s = 0;
    for (int i = 0; i < ctas * kWarps; ++i) s += sh.mass[i];
    cluster_sync();
    return s;
  };

  // ---- the cuts: keys above `cut` stay, and `stay` of those equal to it
  uint32_t cut = 0;
  unsigned long long stay = ~0ull;
  // The largest key up to which, from above, what f(key, logit) counts sums to at least `need`; *rest: what is needed there.  Three
  // rounds of 11, 11 and 10 bits.
  const auto search = [&](unsigned long long need, auto&& f, unsigned long long* rest) {
    uint32_t prefix = 0;
    for (int round = 0; round < 3; ++round) {
      const int shift = round == 0 ? 21 : (round == 1 ? 10 : 0), bits = round == 2 ? 10 : 11;
      for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = 0;
      __syncthreads();
      const uint32_t mask = round == 0 ? 0u : (0xffffffffu << (shift + bits));
      each([&](int, const float4& v) {
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t key = key_of(e[j]);
          if ((key & mask) != prefix) continue;
          const unsigned long long n = f(key, e[j]);
          if (n != 0) atomicAdd(&sh.hist[(key >> shift) & ((1u << bits) - 1u)], n);
        }
      });
      cluster_sync();
      if (rank == 0) {
        // sums of four bins a thread, from the highest on
        const int bin0 = kBins - 4 - 4 * threadIdx.x;
        unsigned long long b[4] = {0, 0, 0, 0}, sum = 0;
        for (int c = 0; c < ctas; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] += ld_cluster_u64(zb_mapa(zb_smem_u32(&sh.hist[bin0 + j]), c));
        sum = b[0] + b[1] + b[2] + b[3];
        unsigned long long upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long u = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += u;
        }
        if (lane == 31) sh.part[warp] = upto;
        __syncthreads();
        unsigned long long before = upto - sum;
        for (int w = 0; w < warp; ++w) before += sh.part[w];
        if (before < need && before + sum >= need) {
          int j = 3;
          while (before + b[j] < need) before += b[j--];
          const uint32_t found = prefix | static_cast<uint32_t>(bin0 + j) << shift;
          for (int c = 0; c < ctas; ++c) {
            st_cluster_u64(zb_mapa(zb_smem_u32(&sh.left), c), need - before);
            st_cluster_u32(zb_mapa(zb_smem_u32(&sh.prefix), c), found);
          }
        }
      }
      cluster_sync();
      prefix = sh.prefix;
      need = sh.left;
    }
    *rest = need;
    return prefix;
  };
  if (top_k == 1) {
    cut = best;
    stay = 1;
  } else {
    if (top_k < p.vocab) cut = search(top_k, [](uint32_t, float) { return 1ull; }, &stay);
    if (top_p < 1.0) {
      unsigned long long above = 0;
      each([&](int, const float4& v) {
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (key_of(e[j]) > cut) above += weight(e[j]);
      });
      above = block_sum(above);
      const unsigned long long at_cut = cut > 0 ? weight(value_of(cut)) : 0;
      const unsigned long long all = above + (cut > 0 ? stay * at_cut : 0);
      const unsigned long long need = min(max(1ull, static_cast<unsigned long long>(ceil(top_p * static_cast<double>(all)))), all);
      if (above >= need) {
        const uint32_t old = cut;
        unsigned long long rest;
        cut = search(need, [&](uint32_t key, float v) { return key > old ? weight(v) : 0ull; }, &rest);
        const unsigned long long w = weight(value_of(cut));
        stay = (rest + w - 1) / w;
      } else {
        stay = (need - above + at_cut - 1) / at_cut;
      }
    }
    if (min_p > 0.0) {
      // the smallest logit whose weight, rounded to 2^-53, is large enough
      const double least = log2(fmin(min_p, 1.0)) - 1.6e-16;
      const float guess = __double2float_ru(fmax(top64 + least / scale, -3.4e38));
      uint32_t k = min(key_of(guess), best);
      const auto fits = [&](uint32_t key) { return key >= best || (static_cast<double>(value_of(key)) - top64) * scale >= least; };
      if (!fits(k)) ++k;
      else if (fits(k - 1)) --k;
      if (k > cut) {
        cut = k;
        stay = ~0ull;
      }
    }
  }

  // ---- what stays, warp after warp
  unsigned long long mass = 0;
  uint32_t ties = 0;
  each([&](int, const float4& v) {
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t key = key_of(e[j]);
      if (key > cut) mass += weight(e[j]);
      ties += key == cut ? 1 : 0;
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane < ctas) {
    st_cluster_u64(zb_mapa(zb_smem_u32(&sh.mass[rank * kWarps + warp]), lane), mass);
    st_cluster_u32(zb_mapa(zb_smem_u32(&sh.ties[rank * kWarps + warp]), lane), ties);
  }
  cluster_sync();
  const unsigned long long tie_weight = cut > 0 ? weight(value_of(cut)) : 0;
  unsigned long long all = 0, before_ties = 0;
  for (int i = 0; i < ctas * kWarps; ++i) {
    const unsigned long long kept = min(static_cast<unsigned long long>(sh.ties[i]), stay - min(stay, before_ties));
    before_ties += sh.ties[i];
    all += sh.mass[i] + kept * tie_weight;
  }
  double u;
  if (p.uniforms == nullptr) u = uniform53(p.rng[0], p.rng[1], row);
  else u = p.uniforms64 ? reinterpret_cast<const double*>(p.uniforms)[row] : static_cast<double>(reinterpret_cast<const float*>(p.uniforms)[row]);
  u = u > 0.0 ? fmin(u, 1.0) : 0.0;                  // NaN: 0
  unsigned long long target = min(static_cast<unsigned long long>(u * static_cast<double>(all)), all - 1);
  before_ties = 0;
  const int me = rank * kWarps + warp;
  unsigned long long sum = 0;
  int owner = 0;
  for (int i = 0; i < ctas * kWarps; ++i) {
    const unsigned long long kept = min(static_cast<unsigned long long>(sh.ties[i]), stay - min(stay, before_ties));
    const unsigned long long here = sh.mass[i] + kept * tie_weight;
    if (sum + here > target) {
      owner = i;
      break;
    }
    sum += here;
    before_ties += sh.ties[i];
  }
  if (owner != me) return;                           // (nobody's shared memory is read from another CTA any more)
  target -= sum;
  unsigned long long tie_room = stay - min(stay, before_ties);
  for (int i = 0; i < rows_of_warp; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(x_s + first + i * 128 + lane * 4);
    const float e[4] = {v.x, v.y, v.z, v.w};
    unsigned long long w[4], mine = 0;
    uint32_t my_ties = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) my_ties += key_of(e[j]) == cut ? 1 : 0;
    uint32_t tie_upto = my_ties;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t n = __shfl_up_sync(0xffffffffu, tie_upto, o);
      if (lane >= o) tie_upto += n;
    }
    unsigned long long tie = tie_upto - my_ties;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t key = key_of(e[j]);
      w[j] = key > cut ? weight(e[j]) : 0ull;
      if (key == cut && tie++ < tie_room) w[j] = tie_weight;
      mine += w[j];
    }
    tie_room -= min(tie_room, static_cast<unsigned long long>(__shfl_sync(0xffffffffu, tie_upto, 31)));
    unsigned long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long n = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += n;
    }
    const unsigned long long row_sum = __shfl_sync(0xffffffffu, upto, 31);
    if (row_sum > target) {
      unsigned long long s = upto - mine;
      if (s <= target && upto > target) {
        int j = 0;
        while (s + w[j] <= target) s += w[j++];
        p.token[row] = from + first + i * 128 + lane * 4 + j;
        if (p.logprob != nullptr)
          p.logprob[row] = e[j] == top ? static_cast<float>(-log(static_cast<double>(all) / kOne))
                                       : static_cast<float>((static_cast<double>(e[j]) - top64) * scale * 0.6931471805599453 - log(static_cast<double>(all) / kOne));
      }
      return;
    }
    target -= row_sum;
  }
}

// CTAs of a row: as many as keep its slices within shared memory, and more while that fills the GPU.
int ctas_of(int rows, int vocab, int sms) {
  int log2 = 0;
  while (log2 < 3 && ((vocab + (1 << log2) - 1) >> log2) > kMaxSlice) ++log2;
  while (log2 < 3 && (static_cast<long long>(rows) << log2) < 2 * sms && (vocab >> log2) > 4 * kThreads) ++log2;
  return log2;
}

template <typename T>
int launch(SampleParams& p, int rows, cudaStream_t s) {
  const int log2 = ctas_of(rows, p.vocab, zb_num_sms()), unit = 128 * kWarps;
  p.slice = ((p.vocab + (1 << log2) - 1) / (1 << log2) + unit - 1) / unit * unit;
  static bool configured[16] = {};
  if (const int rc = zb_config_smem_once(zb_sample_kernel<T>, (kMaxSlice + unit) * 4, configured)) return rc;
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
