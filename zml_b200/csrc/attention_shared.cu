// Attention of single tokens in a batch whose sequences share their first keys (a prompt that is answered many times, an instruction in front of many
// users' questions), bf16, head_dim 64, 128 and 256.
//
// A group of sequences has the same pages in front.  For the keys there, the queries of ALL members and of all heads of a key head are rows of one
// matrix product, and the keys are read once; for the keys behind, the rows are the heads of one sequence.  Either is a list of items - (128 rows, key head, a range
// of keys) - and one kernel walks all of them on the tensor cores (tcgen05, S and O in tensor memory, P as its A operand):
//   S = Q K^T,  m = max S,  P = 2^(S - m),  l = sum P,  O = P V   of every item's range, and
//   o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i,  M = max m_i   over the ranges i that a row was in (zb_shared_merge_kernel).
// What bounds it: the keys' bytes.  A tile of 64 keys of head_dim 128 is 32 KB, 1400 clocks of an SM's share of the memory rate; its products on 128
// rows are 512 clocks whether the rows are in use or not, so that items of four rows need no other kernel.  The line of all items' tiles is cut into
// equal pieces, one for each CTA (two on an SM up to head_dim 128: the hand-overs S -> softmax -> P of one hide under the other's), whatever the
// lengths are; they are read from the device, so that a captured launch serves any lengths and groups.
//   warps 0-3 : softmax and epilogue, one thread a row; they also bring in the rows' queries
//   warp 4    : TMA producer, K and V tiles through a ring that does not stop at the end of an item
//   warp 5    : one thread issues the MMAs
// Every wait is bounded; a wait that runs out records a status and the CTA leaves through its normal exit.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "host_api.h"

int zb_make_tmap_kv_box(CUtensorMap* out, const void* base, long long slots, int kv_heads, int head_dim, int box_rows, int box_subs);

namespace {

constexpr int kRows = 128, kKeys = 64, kThreads = 192;
constexpr uint32_t kKernelId = 42;
constexpr float kLazy = 8.f;                         // a row's reference moves when its maximum has grown by 2^kLazy
constexpr int kMaxBatch = 1024;

struct SharedParams {
  const __nv_bfloat16* q;        // [batch, hq, HD], rows q_stride apart
  const int32_t* block_table;    // [batch, max_pages]
  const int32_t* seq_lens;       // [batch]
  const int32_t* rows;           // [listed]: the groups' members, group after group
  const int32_t* starts;         // [groups + 1]
  const int32_t* lens;           // [groups]: keys that a group shares
  int32_t* where;                // [batch][8], see zb_shared_merge_kernel
  float* part_o;                 // [part_rows(...)][HD]
  float2* part_ml;
  long long q_stride;
  int batch, listed, groups, hkv, group, max_pages, page_size;
  int per_tile;                  // sequences of a tile of 128 rows
  int own_row;                   // the first row of part_o that parts of a sequence's own keys take
  float scale_log2;
  ZbStatus* status;
};

template <int HD>
struct Shape {
  static constexpr int kStages = HD == 64 ? 4 : 2;
  static constexpr int kSubs = HD / 64;
  static constexpr int kQBytes = kRows * HD * 2, kKvBytes = kKeys * HD * 2;
  static constexpr int kTmemCols = HD == 256 ? 512 : 256;
  static constexpr int kCtas = HD == 256 ? 1 : 2;                  // on an SM
  static constexpr uint32_t kColO = 128;                           // S: 0 and 64
  static constexpr int kSmem = kQBytes + 2 * kStages * kKvBytes + 1024 + 256;      // and the plan's numbers
};

// The batch as entries 0 .. groups - 1 (what a group shares) and groups .. groups + batch - 1 (what a sequence has of its own), and the tiles
// of keys of all entries as one line: entry e has those from units[e] on.  An entry's items are its (tile of rows, key head), each `blocks(e)` long.
struct Plan {
  int* starts;                   // [groups + 1], clamped
  int* end;                      // [entries]: keys [begin, end) of an entry
  int* begin;                    // [batch]
  int* units;                    // [entries + 1]
  int groups, entries;
  ZB_DEVICE int group_of(int i) const {               // of the i-th of `rows`, -1: none
    int lo = 0, hi = groups;                         // the last group that starts at or in front of i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= i) lo = mid; else hi = mid;
    }
    return groups > 0 && i >= starts[lo] && i < starts[lo + 1] ? lo : -1;
  }
  ZB_DEVICE int blocks(int e) const { return (end[e] + kKeys - 1) / kKeys - (e < groups ? 0 : begin[e - groups] / kKeys); }
};

struct Segment {                 // the part of an item that a CTA works on
  int entry, tile, head;
  int block, count;              // tiles of 64 keys, from key 64 * block on
};

struct Walk {
  int at, to, entry;
  ZB_DEVICE void start(const Plan& p, int from, int until) {
    at = from;
    to = until;
    int lo = 0, hi = p.entries;                      // the last entry with units[entry] <= from
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.units[mid] <= from) lo = mid; else hi = mid;
    }
    entry = lo;
  }
  ZB_DEVICE bool next(const Plan& p, int hkv, Segment& s) {
    if (at >= to) return false;
    while (p.units[entry + 1] <= at) ++entry;
    const int n = p.blocks(entry), local = at - p.units[entry], item = local / n, j = local - item * n;
    s.entry = entry;
    s.tile = item / hkv;
    s.head = item - s.tile * hkv;
    s.count = min(n - j, to - at);
    s.block = j + (entry < p.groups ? 0 : p.begin[entry - p.groups] / kKeys);
    at += s.count;
    return true;
  }
};

// max of three, one instruction
ZB_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// First tile of CTA c of n, of `total` tiles; and the CTA that has tile u.
ZB_DEVICE int first_of(int c, int n, int total) { return static_cast<int>(static_cast<long long>(total) * c / n); }
ZB_DEVICE int owner_of(int u, int n, int total) { return static_cast<int>((static_cast<long long>(u + 1) * n - 1) / total); }

ZB_DEVICE int clamp_keys(int n, const SharedParams& p) { return min(max(n, 0), p.max_pages * p.page_size); }

// All threads of the CTA.  Returns the number of tiles of the line.
ZB_DEVICE int make_plan(const SharedParams& p, Plan& plan, long long* scratch) {
  const int g_n = p.groups, e_n = g_n + p.batch, tid = threadIdx.x;
  for (int g = tid; g <= g_n; g += kThreads) plan.starts[g] = min(max(p.starts[g], 0), p.listed);
  for (int b = tid; b < p.batch; b += kThreads) {
    plan.begin[b] = 0;
    plan.end[g_n + b] = clamp_keys(p.seq_lens[b], p);
  }
  for (int g = tid; g < g_n; g += kThreads) plan.end[g] = clamp_keys(p.lens[g], p);
  __syncthreads();
  for (int i = tid; i < p.listed; i += kThreads) {
    const int g = plan.group_of(i), b = p.rows[i];
    if (g >= 0 && b >= 0 && b < p.batch) plan.begin[b] = plan.end[g];
  }
  __syncthreads();
  // sums up to every entry: a run of entries a thread, then threads, then warps
  const int each = (e_n + kThreads - 1) / kThreads, e0 = min(tid * each, e_n), e1 = min(e0 + each, e_n);
  const auto count = [&](int e) {
    if (e >= g_n) return plan.end[e] > plan.begin[e - g_n] ? static_cast<long long>(p.hkv) * plan.blocks(e) : 0ll;
    return static_cast<long long>((max(plan.starts[e + 1] - plan.starts[e], 0) + p.per_tile - 1) / p.per_tile) * p.hkv * plan.blocks(e);
  };
  long long mine = 0;
  for (int e = e0; e < e1; ++e) mine += count(e);
  long long upto = mine;
  const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) scratch[warp] = upto;
  __syncthreads();
  long long before = upto - mine, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  for (int e = e0; e < e1; ++e) {
    plan.units[e] = static_cast<int>(before);
    before += count(e);
  }
  if (tid == 0) plan.units[e_n] = static_cast<int>(total);
  __syncthreads();
  if (total > 0x3fffffffll) {                        // groups that overlap many times over
    if (tid == 0) zb_record_error(p.status, ZB_ERR_BAD_ARG, kKernelId, 20u, static_cast<uint32_t>(total >> 10));
    return 0;
  }
  return static_cast<int>(total);
}

template <int HD>
__global__ void __launch_bounds__(kThreads, Shape<HD>::kCtas)
zb_shared_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const SharedParams p) {
  using S = Shape<HD>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* q_s = smem;
  uint8_t* k_s = q_s + S::kQBytes;                   // [kStages][kKvBytes]
  uint8_t* v_s = k_s + kStages * S::kKvBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + kStages * S::kKvBytes);
  uint64_t* q_full = bars;                           // four warps
  uint64_t* k_full = bars + 1;                       // kStages
  uint64_t* v_full = k_full + kStages;               // kStages
  uint64_t* k_empty = v_full + kStages;              // kStages: S of the tile is done
  uint64_t* v_empty = k_empty + kStages;             // kStages: so is O
  uint64_t* s_full = v_empty + kStages;              // two buffers
  uint64_t* p_full = s_full + 2;                     // two buffers, four warps
  uint64_t* o_ready = p_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(o_ready + 1);
  volatile uint32_t* abort_flag = tmem_holder + 1;
  volatile uint32_t* abort_where = tmem_holder + 2;
  Plan plan;
  plan.groups = p.groups;
  plan.entries = p.groups + p.batch;
  plan.starts = reinterpret_cast<int*>(bars + 32);
  plan.end = plan.starts + p.groups + 1;
  plan.begin = plan.end + plan.entries;
  plan.units = plan.begin + p.batch;
  __shared__ long long scratch[kThreads / 32];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    zb_mbar_init(q_full, 4);
    for (int s = 0; s < kStages; ++s) {
      zb_mbar_init(&k_full[s], 1);
      zb_mbar_init(&v_full[s], 1);
      zb_mbar_init(&k_empty[s], 1);
      zb_mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      zb_mbar_init(&s_full[i], 1);
      zb_mbar_init(&p_full[i], 4);
    }
    zb_mbar_init(o_ready, 1);
    *abort_flag = 0u;
    *abort_where = 0u;
    zb_mbar_fence_init();
    zb_tma_prefetch_desc(&tmap_k);
    zb_tma_prefetch_desc(&tmap_v);
  }
  if (warp == 5) {
    zb_tmem_alloc(tmem_holder, S::kTmemCols);
    zb_tmem_relinquish();
  }
  zb_pdl_wait();                                     // the batch description, queries and keys come from preceding work
  const int total = make_plan(p, plan, scratch), ctas = min(static_cast<int>(gridDim.x), total);      // that have a tile
  zb_tc_fence_before();
  __syncthreads();
  zb_tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  zb_pdl_launch();                                   // only now: a successor that also takes tensor memory must not come first

  // For zb_shared_merge_kernel: where a sequence's parts are.
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < p.batch; b += kThreads) {
      const int e = p.groups + b;
      const bool some = total > 0 && plan.units[e + 1] > plan.units[e];
      reinterpret_cast<int4*>(p.where)[2 * b] = make_int4(0, 0, 0, 0);
      reinterpret_cast<int4*>(p.where)[2 * b + 1] = make_int4(some ? plan.blocks(e) : 0, plan.units[e], total, 0);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.listed; i += kThreads) {
      const int g = plan.group_of(i), b = p.rows[i];
      if (g < 0 || b < 0 || b >= p.batch || total == 0 || plan.units[g + 1] == plan.units[g]) continue;
      const int n = plan.blocks(g), at = i - plan.starts[g], tile = at / p.per_tile, first = plan.starts[g] + tile * p.per_tile;
      reinterpret_cast<int4*>(p.where)[2 * b] =
          make_int4(n, plan.units[g] + tile * p.hkv * n, first * p.hkv + i - first, min(p.per_tile, plan.starts[g + 1] - first));
    }
  }

  const int cta = blockIdx.x, from = cta < ctas ? first_of(cta, ctas, total) : 0, to = cta < ctas ? first_of(cta + 1, ctas, total) : 0;
  Walk walk;
  Segment seg;
  if (from < to) walk.start(plan, from, to); else walk.at = walk.to = 0;

  if (warp == 4) {
    // ------------------------------------------------------------------ TMA producer
    // Pages of 64 tokens and more come as one box of all columns; of smaller ones several make up a tile, a box each and 64 columns.
    const int box = min(p.page_size, kKeys), pages_of_tile = kKeys / box;
    uint32_t stage = 0, phase = 0;
    int done = 0;
    bool ok = true;
    while (ok && walk.next(plan, p.hkv, seg)) {
      int seq;
      if (seg.entry >= p.groups) {
        seq = seg.entry - p.groups;
      } else {                                       // any member's pages are the group's
        seq = 0;
        for (int i = plan.starts[seg.entry]; i < plan.starts[seg.entry + 1]; ++i) {
          seq = p.rows[i];
          if (seq >= 0 && seq < p.batch) break;
          seq = 0;
        }
      }
      const int32_t* table = p.block_table + static_cast<size_t>(seq) * p.max_pages;
      const int end = plan.end[seg.entry];
      for (int j0 = 0; ok && j0 < seg.count; j0 += 32 / pages_of_tile) {
        // a lane for each box: its first slot of the cache; behind the end it lies outside of the cache, which reads as zeros
        const int key = (seg.block + j0) * kKeys + lane * box;
        int slot = -kKeys;
        if (key < end && (j0 + lane / pages_of_tile) < seg.count) {
          const int page = table[key / p.page_size];
          if (ZB_BC_OK(page, ZB_BC_PAGES, kKernelId, 1) && page >= 0) slot = page * p.page_size + key % p.page_size;
        }
        const int n = min(seg.count - j0, 32 / pages_of_tile);
        for (int j = 0; j < n; ++j) {
          // K, then V: a tile's K is done with two tiles before its V is
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint64_t *full = w == 0 ? &k_full[stage] : &v_full[stage], *empty = w == 0 ? &k_empty[stage] : &v_empty[stage];
            if (done >= kStages && !__all_sync(0xffffffffu, zb_mbar_wait(empty, phase ^ 1u, abort_flag))) {
              *abort_where = 1u;
              ok = false;
              break;
            }
            uint8_t* dst = (w == 0 ? k_s : v_s) + stage * S::kKvBytes;
            const CUtensorMap* map = w == 0 ? &tmap_k : &tmap_v;
            if (lane == 0) zb_mbar_expect_tx(full, S::kKvBytes);
            __syncwarp();
            if (pages_of_tile == 1) {
              const int at = __shfl_sync(0xffffffffu, slot, j);
              if (lane == 0) zb_tma_load_4d(dst, map, full, 0, at, 0, seg.head);
            } else {
              const int i = lane - j * pages_of_tile;
              if (i >= 0 && i < pages_of_tile) {
#pragma unroll
                for (int c = 0; c < S::kSubs; ++c) zb_tma_load_4d(dst + c * (kKeys * 128) + i * box * 128, map, full, 0, slot, c, seg.head);
              }
            }
          }
          if (!ok) break;
          ++done;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t kIdescS = zb_make_idesc_bf16(kRows, kKeys);
      constexpr uint32_t kIdescO = zb_make_idesc_bf16(kRows, HD) | (1u << 16);         // B (= V) is MN-major
      const uint32_t t_s = tmem_base, t_o = tmem_base + S::kColO, qa = zb_smem_u32(q_s);
      uint32_t k_stage = 0, k_phase = 0, stage = 0, phase = 0, where = 0;
      int s_done = 0, done = 0, segment = 0;
      // S of the next tile, into the buffer that is its number's parity
      const auto next_s = [&]() {
        if (!zb_mbar_wait(&k_full[k_stage], k_phase, abort_flag)) return false;
        zb_tc_fence_after();
        const uint32_t ka = zb_smem_u32(k_s + k_stage * S::kKvBytes);
        const int b = s_done & 1;
#pragma unroll
        for (int c = 0; c < S::kSubs; ++c) {
          const uint64_t dq = zb_make_desc_sw128(qa + c * (kRows * 128)), dk = zb_make_desc_sw128(ka + c * (kKeys * 128));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) zb_umma_f16(t_s + b * kKeys, dq + 2 * kk, dk + 2 * kk, kIdescS, (c > 0 || kk > 0) ? 1u : 0u);
        }
        zb_umma_commit(&s_full[b]);
        zb_umma_commit(&k_empty[k_stage]);
        ++s_done;
        if (++k_stage == kStages) {
          k_stage = 0;
          k_phase ^= 1u;
        }
        return true;
      };
      while (where == 0u && walk.next(plan, p.hkv, seg)) {
        if (!zb_mbar_wait(q_full, static_cast<uint32_t>(segment) & 1u, abort_flag)) {
          where = 2u;
          break;
        }
        ++segment;
        if (!next_s() || (seg.count > 1 && !next_s())) {
          where = 3u;
          break;
        }
        for (int j = 0; j < seg.count; ++j) {
          if (!zb_mbar_wait(&v_full[stage], phase, abort_flag)) {
            where = 4u;
            break;
          }
          if (!zb_mbar_wait(&p_full[done & 1], static_cast<uint32_t>(done >> 1) & 1u, abort_flag)) {
            where = 5u;
            break;
          }
          zb_tc_fence_after();
          // O (+)= P V: steps of 16 keys; A = P in tensor memory (8 columns per step), B = V, MN-major
          const uint32_t va = zb_smem_u32(v_s + stage * S::kKvBytes);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            zb_umma_f16_ts(t_o, t_s + (done & 1) * kKeys + 8 * k, zb_make_desc_sw128_mn(va + k * (16 * 128), kKeys * 128, 1024), kIdescO,
                           (j > 0 || k > 0) ? 1u : 0u);
          zb_umma_commit(o_ready);
          zb_umma_commit(&v_empty[stage]);
          if (j + 2 < seg.count && !next_s()) {       // over P, in order behind the MMAs that read it
            where = 6u;
            break;
          }
          ++done;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (where != 0u) *abort_where = where;
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue (one row per thread)
    const int r = warp * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t t_o = tmem_base + S::kColO + lane_off;
    const ZbF2 sc2 = zb_pack2(p.scale_log2, p.scale_log2);
    int it = 0;                                      // tiles so far
    bool ok = true;
    while (ok && walk.next(plan, p.hkv, seg)) {
      // ---- the item's rows: row i is head i % group of its sequence i / group
      const bool common = seg.entry < p.groups;
      const int first = common ? plan.starts[seg.entry] + seg.tile * p.per_tile : 0;
      const int seqs = common ? min(p.per_tile, plan.starts[seg.entry + 1] - first) : 1, rows = seqs * p.group;
      const int end = plan.end[seg.entry], lo = common ? 0 : plan.begin[seg.entry - p.groups];
      const bool mine = warp * 32 < rows;            // the warp has rows at all
      const int row = min(r, rows - 1);              // lanes behind the last row repeat it
      int limit = end;
      if (mine) {
        const int n = row / p.group;
        int seq = common ? p.rows[first + n] : seg.entry - p.groups;
        if (seq < 0 || seq >= p.batch) {
          seq = 0;
          limit = 0;
        }
        if (common) limit = min(limit, plan.end[p.groups + seq]);
        // 16 bytes at a time, neighbouring lanes a row's neighbouring pieces
        const long long at = seq * p.q_stride + (seg.head * p.group + row - n * p.group) * HD;
        constexpr int kPieces = HD / 8, kOnce = 32 / kPieces > 0 ? 32 / kPieces : 1;
#pragma unroll 4
        for (int i = 0; i < 32; i += kOnce) {
          const int src = i + lane / kPieces, piece = lane % kPieces, to_row = warp * 32 + src;
          const long long from_at = __shfl_sync(0xffffffffu, at, src);
          const uint4 x = *reinterpret_cast<const uint4*>(p.q + from_at + piece * 8);
          *reinterpret_cast<uint4*>(q_s + (piece >> 3) * (kRows * 128) + to_row * 128 + (((piece & 7) ^ (to_row & 7)) << 4)) = x;
        }
        zb_fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) zb_mbar_arrive(q_full);
      const int least = __reduce_min_sync(0xffffffffu, limit);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < seg.count; ++j, ++it) {
        const int b = it & 1;
        const uint32_t t_s = tmem_base + b * kKeys + lane_off;
        if (!__all_sync(0xffffffffu, zb_mbar_wait(&s_full[b], static_cast<uint32_t>(it >> 1) & 1u, abort_flag))) {
          *abort_where = 10u;
          ok = false;
          break;
        }
        const int key0 = (seg.block + j) * kKeys;
        if (mine) {
          zb_tc_fence_after();
          uint32_t sr[64];
          zb_tmem_ld32(t_s, reinterpret_cast<uint32_t(&)[32]>(sr[0]));
          zb_tmem_ld32(t_s + 32, reinterpret_cast<uint32_t(&)[32]>(sr[32]));
          zb_tmem_ld_wait();
          if (key0 + kKeys > least || key0 < lo) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (key0 + i >= limit || key0 + i < lo) sr[i] = 0xff800000u;                        // -inf
          }
          float mx4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mx4[i] = __uint_as_float(sr[i]);
#pragma unroll
          for (int i = 4; i < 60; i += 2) mx4[(i >> 1) & 3] = max3(mx4[(i >> 1) & 3], __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
          mx4[0] = max3(mx4[0], __uint_as_float(sr[60]), __uint_as_float(sr[61]));
          mx4[1] = max3(mx4[1], __uint_as_float(sr[62]), __uint_as_float(sr[63]));
          const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]) * p.scale_log2;              // in units of log2
          float alpha = 1.f;
          if (mx > m + kLazy) {                      // also the first visible key: m = -inf
            alpha = m == -INFINITY ? 1.f : zb_ex2(m - mx);
            m = mx;
            l *= alpha;
          }
          if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            // O += P V of the previous tile must be complete (that of the one before it is: S of this tile went behind it)
            if (!__all_sync(0xffffffffu, zb_mbar_wait(o_ready, static_cast<uint32_t>(it - 1) & 1u, abort_flag))) {
              *abort_where = 11u;
              ok = false;
              break;
            }
            zb_tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 16) {
              uint32_t o[16];
              zb_tmem_ld16(t_o + c0, o);
              zb_tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              zb_tmem_st16(t_o + c0, o);
            }
          }
          // p = 2^(s * scale - m)
          const float neg_m = m == -INFINITY ? 0.f : -m;
          const ZbF2 nm2 = zb_pack2(neg_m, neg_m);
          ZbF2 sum[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pw[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int e = 32 * c + 2 * i;
              float x0, x1;
              zb_unpack2(zb_fma2(zb_pack2(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1])), sc2, nm2), x0, x1);
              x0 = zb_ex2(x0);
              x1 = zb_ex2(x1);
              pw[i] = zb_pack_bf16x2(x0, x1);
              sum[i & 1] = zb_add2(sum[i & 1], zb_pack2(x0, x1));
            }
            zb_tmem_st16(t_s + 16 * c, pw);
          }
          l += zb_sum2(zb_add2(sum[0], sum[1]));
        }
        // Rows of V behind the end of the keys hold whatever was there before, perhaps NaN, which a weight of zero does not make zero: they are
        // cleared in shared memory, a warp 16 rows of the tile.
        if (key0 + kKeys > end) {
          const int stage = it % kStages;
          if (!__all_sync(0xffffffffu, zb_mbar_wait(&v_full[stage], static_cast<uint32_t>(it / kStages) & 1u, abort_flag))) {
            *abort_where = 12u;
            ok = false;
            break;
          }
          uint4* v = reinterpret_cast<uint4*>(v_s + stage * S::kKvBytes);                         // the swizzle stays within a row of 128 bytes
          for (int c = 0; c < S::kSubs; ++c)
            for (int i = warp * 128 + lane; i < (warp + 1) * 128; i += 32)
              if (key0 + (i >> 3) >= end) v[c * kKeys * 8 + i] = make_uint4(0u, 0u, 0u, 0u);
          zb_fence_proxy_async_smem();
        }
        // Parity does not tell a phase of o_ready from the one two before it, so that no wait may begin two phases early or end two late: the
        // last tile but one is waited for while the last one is still held back.
        if (j > 0 && j == seg.count - 1 && !__all_sync(0xffffffffu, zb_mbar_wait(o_ready, static_cast<uint32_t>(it - 1) & 1u, abort_flag))) {
          *abort_where = 13u;
          ok = false;
          break;
        }
        zb_tmem_st_wait();
        zb_tc_fence_before();
        __syncwarp();
        if (lane == 0) zb_mbar_arrive(&p_full[b]);
      }
      if (!ok) break;
      if (!__all_sync(0xffffffffu, zb_mbar_wait(o_ready, static_cast<uint32_t>(it - 1) & 1u, abort_flag))) {
        *abort_where = 14u;
        ok = false;
        break;
      }
      if (mine) {
        zb_tc_fence_after();
        // rows of parts, disjoint: an item's own, and as many again for every CTA in front
        const long long at = (common ? (static_cast<long long>(first) * p.hkv + seg.head * seqs) * p.group + static_cast<long long>(blockIdx.x) * kRows
                                     : p.own_row + (static_cast<long long>(seg.entry - p.groups) * p.hkv + seg.head + blockIdx.x) * p.group) + r;
        float* dst = p.part_o + at * HD;
        if (r < rows) p.part_ml[at] = make_float2(m, l);
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += 32) {
          uint32_t o[32];
          zb_tmem_ld32(t_o + c0, o);
          zb_tmem_ld_wait();
          if (r < rows) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(dst + c0 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        zb_tc_fence_before();                        // the next item's MMAs write O again behind q_full
      }
    }
  }

  // ------------------------------------------------------------------ common exit
  zb_tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0u) {
    if (threadIdx.x == 0) zb_record_error(p.status, ZB_ERR_MBAR_TIMEOUT, kKernelId, *abort_where, blockIdx.x);
    const uint64_t t0 = zb_globaltimer();            // copies still in flight must land before the shared memory is reused
    while (zb_globaltimer() - t0 < 200000ull) {
    }
    __syncthreads();
  }
  if (warp == 5) {
    zb_tc_fence_after();
    zb_tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// The rows of one (sequence, key head): a warp for each, over all parts that the kernel above left of it.  where[seq] = {tiles of the prefix, first of them
// (of key head 0), row of its parts in units of `group` (likewise), step of these to the next key head; tiles of its own, first of them, tiles of the line}.
template <int HD>
__global__ void __launch_bounds__(128)
zb_shared_merge_kernel(const int32_t* __restrict__ where, const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                       __nv_bfloat16* __restrict__ out, int hkv, int group, int own_row, int part_rows, int ctas) {
  constexpr int kEach = HD / 32;
  zb_pdl_launch();
  zb_pdl_wait();
  const int b = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 front = reinterpret_cast<const int4*>(where)[2 * b], back = reinterpret_cast<const int4*>(where)[2 * b + 1];
  const int total = back.z;
  ctas = min(ctas, total);
  int n0 = 0, n1 = 0, c0 = 0, c1 = 0;
  if (front.x > 0) {
    const int u = front.y + head * front.x;
    c0 = owner_of(u, ctas, total);
    n0 = owner_of(u + front.x - 1, ctas, total) - c0 + 1;
  }
  if (back.x > 0) {
    const int u = back.y + head * back.x;
    c1 = owner_of(u, ctas, total);
    n1 = owner_of(u + back.x - 1, ctas, total) - c1 + 1;
  }
  const int n = n0 + n1;
  for (int r = warp; r < group; r += 4) {
    const long long row0 = (static_cast<long long>(front.z) + static_cast<long long>(head) * front.w) * group + static_cast<long long>(c0) * kRows + r;
    const long long row1 = own_row + (static_cast<long long>(b) * hkv + head + c1) * group + r;
    const auto place = [&](int i) {                  // (a sequence that is in two groups finds a wrong row, but one that is there)
      const long long at = i < n0 ? row0 + static_cast<long long>(i) * kRows : row1 + static_cast<long long>(i - n0) * group;
      return at < part_rows ? at : 0ll;
    };
    float acc[kEach], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int j = 0; j < kEach; ++j) acc[j] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int most = min(32, n - i0);
      const float2 ml = lane < most ? part_ml[place(i0 + lane)] : make_float2(-INFINITY, 0.f);
      const float up = fmaxf(top, zb_warp_max(ml.x)), base = up == -INFINITY ? 0.f : up;
      const float was = zb_ex2(top - base), f = zb_ex2(ml.x - base);
      top = up;
      sum = sum * was + zb_warp_sum(f * ml.y);
#pragma unroll
      for (int j = 0; j < kEach; ++j) acc[j] *= was;
#pragma unroll 4
      for (int i = 0; i < most; ++i) {
        const float by = __shfl_sync(0xffffffffu, f, i);
        const float* src = part_o + place(i0 + i) * HD + lane * kEach;
#pragma unroll
        for (int j = 0; j < kEach; ++j) acc[j] += by * src[j];
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no key at all: zeros
    __nv_bfloat16* dst = out + (static_cast<size_t>(b) * hkv * group + head * group + r) * HD + lane * kEach;
#pragma unroll
    for (int j = 0; j < kEach; j += 2) *reinterpret_cast<uint32_t*>(dst + j) = zb_pack_bf16x2(acc[j] * inv, acc[j + 1] * inv);
  }
}

int plan_bytes(int batch, int groups) { return 4 * (groups + 1 + (groups + batch) + batch + groups + batch + 1); }

// CTAs of the walk: as many as fit at once.
template <int HD>
int walk_ctas(int batch, int groups, int sms) {
  const int smem = Shape<HD>::kSmem + plan_bytes(batch, groups);
  return sms * (Shape<HD>::kCtas == 2 && 2 * (smem + 1024) <= 228 * 1024 ? 2 : 1);
}
int walk_ctas(int hd, int batch, int groups, int sms) {
  return hd == 64 ? walk_ctas<64>(batch, groups, sms) : hd == 128 ? walk_ctas<128>(batch, groups, sms) : walk_ctas<256>(batch, groups, sms);
}

// Rows of the parts: of prefixes (from row 0 on) and of the sequences' own keys.
long long prefix_rows(int listed, int hq, int ctas) { return static_cast<long long>(listed) * hq + static_cast<long long>(ctas) * kRows; }
long long part_rows(int listed, int batch, int hq, int group, int ctas) {
  return (prefix_rows(listed, hq, ctas) + static_cast<long long>(batch) * hq + static_cast<long long>(ctas) * group + 1) & ~1ll;      // (16 bytes)
}

template <int HD>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const SharedParams& p, void* out, int rows, int ctas, cudaStream_t s) {
  static bool configured[16] = {};
  if (const int rc = zb_config_smem_once(zb_shared_decode_kernel<HD>, Shape<HD>::kSmem + plan_bytes(kMaxBatch, kMaxBatch), configured)) return rc;
  cudaError_t e = zb_launch(zb_shared_decode_kernel<HD>, dim3(ctas), dim3(kThreads), Shape<HD>::kSmem + plan_bytes(p.batch, p.groups), s, tk, tv, p);
  if (e == cudaSuccess)
    e = zb_launch(zb_shared_merge_kernel<HD>, dim3(p.batch, p.hkv), dim3(128), 0, s, p.where, p.part_o, p.part_ml, reinterpret_cast<__nv_bfloat16*>(out),
                  p.hkv, p.group, p.own_row, rows, ctas);
  zb_count_launch(2);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

bool takes(int batch, int listed, int groups, int hq, int hkv, int hd, int page_size) {
  return batch > 0 && batch <= kMaxBatch && listed >= 0 && listed <= batch && groups >= 0 && groups <= batch && hkv > 0 && hkv <= 65535 && hq > 0 &&
         hq % hkv == 0 && hq / hkv <= kRows && (hd == 64 || hd == 128 || hd == 256) && (page_size == 16 || page_size == 32 || (page_size > 0 && page_size % kKeys == 0));
}

}  // namespace

extern "C" {

// Bytes of a call's workspace, which needs no particular contents; 0: sizes that the kernel does not take.
long long zb_shared_decode_workspace(int batch, int listed, int groups, int hq, int hkv, int hd, int page_size) {
  ZbDeviceState* st = zb_device_state();
  if (!st || !takes(batch, listed, groups, hq, hkv, hd, page_size)) return 0;
  return 32ll * batch + 4 * (hd + 2) * part_rows(listed, batch, hq, hq / hkv, walk_ctas(hd, batch, groups, st->num_sms));
}

// The arguments of a call, as the caller packs them (ops/shared.py).
struct ZbSharedDecode {
  const void* q;                                   // [batch, hq, hd], rows on 16 bytes
  const void *k_cache, *v_cache;                   // [pages, page_size, hkv, hd], contiguous, on 16 bytes
  void* out;                                       // [batch, hq, hd], contiguous, on 4 bytes
  const int32_t* block_table;                      // [batch, max_pages]
  const int32_t* seq_lens;                         // [batch]
  const int32_t* rows;                             // [listed]
  const int32_t* starts;                           // [groups + 1]
  const int32_t* lens;                             // [groups]
  void* work;                                      // what zb_shared_decode_workspace asked for, on 32 bytes
  void* stream;
  long long q_stride;
  int batch, listed, groups, hq, hkv, hd, page_size, max_pages, num_pages;
  float scale;
};

int zb_shared_decode(const ZbSharedDecode* c) {
  if (c->batch <= 0) return 0;
  if (!takes(c->batch, c->listed, c->groups, c->hq, c->hkv, c->hd, c->page_size)) return -30;
  const long long keys = static_cast<long long>(c->max_pages) * c->page_size, slots = static_cast<long long>(c->num_pages) * c->page_size;
  // (tiles of the line: 32 bits)
  if (c->max_pages <= 0 || slots <= 0 || slots > 0x7fffff00ll || keys > 0x7fffff00ll || 2ll * c->batch * c->hkv * ((keys + kKeys - 1) / kKeys) > 0x3fffffffll) return -31;
  if (((reinterpret_cast<uintptr_t>(c->q) | reinterpret_cast<uintptr_t>(c->k_cache) | reinterpret_cast<uintptr_t>(c->v_cache)) & 15) != 0 || c->q_stride % 8 != 0 ||
      (reinterpret_cast<uintptr_t>(c->out) & 3) != 0 || (reinterpret_cast<uintptr_t>(c->work) & 31) != 0)
    return -32;
  if (!(c->scale > 0.f)) return -33;
  ZbDeviceState* st = zb_device_state();
  if (!st) return -20;
  const int group = c->hq / c->hkv, ctas = walk_ctas(c->hd, c->batch, c->groups, st->num_sms), box = std::min(c->page_size, kKeys);
  const int subs = box < kKeys ? 1 : c->hd / 64;
  const long long rows = part_rows(c->listed, c->batch, c->hq, group, ctas);
  if (rows > 0x7fffffffll) return -34;
  CUtensorMap tk, tv;
  int rc = zb_make_tmap_kv_box(&tk, c->k_cache, slots, c->hkv, c->hd, box, subs);
  if (rc == 0) rc = zb_make_tmap_kv_box(&tv, c->v_cache, slots, c->hkv, c->hd, box, subs);
  if (rc != 0) return rc;
  SharedParams p = {};
  p.q = reinterpret_cast<const __nv_bfloat16*>(c->q);
  p.block_table = c->block_table;
  p.seq_lens = c->seq_lens;
  p.rows = c->rows;
  p.starts = c->starts;
  p.lens = c->lens;
  p.where = reinterpret_cast<int32_t*>(c->work);
  p.part_ml = reinterpret_cast<float2*>(p.where + 8 * c->batch);
  p.part_o = reinterpret_cast<float*>(p.part_ml + rows);
  p.q_stride = c->q_stride;
  p.batch = c->batch;
  p.listed = c->listed;
  p.groups = c->groups;
  p.hkv = c->hkv;
  p.group = group;
  p.max_pages = c->max_pages;
  p.page_size = c->page_size;
  p.per_tile = kRows / group;
  p.own_row = static_cast<int>(prefix_rows(c->listed, c->hq, ctas));
  p.scale_log2 = c->scale * 1.4426950408889634f;
  p.status = st->status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(c->stream);
  const int n = static_cast<int>(rows);
  if (c->hd == 64) return launch<64>(tk, tv, p, c->out, n, ctas, s);
  return c->hd == 128 ? launch<128>(tk, tv, p, c->out, n, ctas, s) : launch<256>(tk, tv, p, c->out, n, ctas, s);
}

}  // extern "C"
