// Attention of single tokens in a batch whose sequences share their first keys (a prompt that is answered many times, an instruction in front of many
// users' questions), bf16, head_dim 64, 128 and 256.
//
// A group of sequences has the same pages in front.  For the keys there, the queries of ALL members and of all heads of a key head are rows of one
// matrix product, and the keys are read once; for the keys behind, the rows are the heads of one sequence.  Either way
//   S = Q K^T,  m = max S,  P = 2^(S - m),  l = sum P,  O = P V   of a range of keys, and
//   o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i,  M = max m_i   over the ranges i that a row was in (zb_shared_merge_kernel).
// Groups' keys: items of (128 rows, key head), tiles of 64 keys on the tensor cores (tcgen05, S and O in tensor memory, P as its A operand).
// Sequences' own keys: items of (sequence, key head), steps of 16 keys by single warps ("walkers") with mma.sync, S^T = K Q^T and O^T = V^T P^T, where up to 8 or 16 heads are
// the columns: 128 rows for four heads took 0.5 us a tile of an SM, and 128 sequences of their own keys twice as long.  (More than 16 heads to a key head: tiles, too.)
// What bounds it: the keys' bytes, and of a long prefix that is shared by more than 128 rows the tiles' chain S -> softmax -> P -> O on two CTAs of an SM (tensor cores and
// exponentials two fifths of the time each).  Either list of items is a line of units that is cut into equal pieces, one for each CTA (two on an SM up to head_dim 128: the
// hand-overs of one hide under the other's) or walker, whatever the lengths are; they are read from the device, so that a captured launch serves any lengths and groups.
//   CTAs of the groups' line     warps 0-3 : softmax and epilogue, one thread a row; they also bring in the rows' queries
//                                warp 4    : TMA producer, K and V tiles through rings that do not stop at the end of an item
//                                warp 5    : one thread issues the MMAs
//   CTAs of the sequences' line  warps 0-5 : walkers, each with a ring of its own that it fills itself
// Measured, calls in a row on other tensors each (beside the bytes' floor): 8 sequences behind 2000 keys, 32 / 8 heads of 128, 18.9 us (1.4; latency: launch, plan, two
// kernels); 32 behind 8192, 32 / 8 heads of 64, 27 (5.2); 128 behind 4133 with 782 own keys on average, 32 / 4 heads of 128, 62 (33: 3.4 TB/s); 64 behind 65536, 32 / 8 heads of
// 128, 120 (47: 575 TFLOP/s; 103 where a graph of a dozen calls is all that runs); 64 behind 8192, 32 heads to one key head of 128, 31 (5.4).
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
constexpr int kStep = 16, kWalkers = 6;
// What counts of a CTA's time.  A tile of a group's keys takes 1.7 - 2.8 us and the six walkers' step 1.05 - 1.7 us; an item's end and the next one's
// beginning (its rows' parts written, other queries, an empty pipe) several of either.  With 7 and 1 instead, the CTAs that crossed items and those of the groups came in last:
// 83 and 130 us where it was 72 and 105 (128 sequences behind 4133 keys, 64 behind 65536; graphs of calls, all heads with the same numbers).
constexpr uint32_t kTileCost = 11;                   // of a tile of a group's keys, in steps of sequences' own
constexpr int kSwitch = 6;                           // of a change of items, in tiles or steps
constexpr int kLeast = 3;                            // tiles of a piece, so that few pieces are none but a change
constexpr int kLeastSteps = 8;                       // steps of a piece: three sequences of 8700 own keys in 400 parts each were merged for 40 us

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
  static constexpr int kTiles = kQBytes + 2 * kStages * kKvBytes;
  static constexpr int kStepBytes = 2 * kStep * HD * 2;            // K and V of a step
  static constexpr int kDepth = kTiles / (kWalkers * kStepBytes);  // steps of a walker's ring
  static constexpr int kSmem = kTiles + 1024 + 512;                // and the plan's numbers
};

// The batch as entries 0 .. groups - 1 (what a group shares) and groups .. groups + batch - 1 (what a sequence has of its own).  An entry's items are
// its (tile of rows, key head), each kSwitch + `blocks(e)` units long - blocks of keys, and what it takes to go from one item to the next.  The units of
// all groups are one line, those of all sequences another, each cut evenly among its CTAs (`Lines`); entry e has those from units[e] on of its line.
template <bool SPLIT>                                // whether sequences' own keys are taken in steps of 16 by single warps, or in tiles of 64
struct Plan {
  int* starts;                   // [groups + 1], clamped
  int* end;                      // [entries]: keys [begin, end) of an entry
  int* begin;                    // [batch]
  int* units;                    // [entries + 2]: of the groups and their sum, then of the sequences and theirs
  int* rows;                     // [listed], -1 for what is no sequence
  int groups, entries;
  ZB_DEVICE int group_of(int i) const {               // of the i-th of `rows`, -1: none
    int lo = 0, hi = groups;                         // the last group that starts at or in front of i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= i) lo = mid; else hi = mid;
    }
    return groups > 0 && i >= starts[lo] && i < starts[lo + 1] ? lo : -1;
  }
  ZB_DEVICE int block_keys(int e) const { return SPLIT && e >= groups ? kStep : kKeys; }
  ZB_DEVICE int first_block(int e) const { return e < groups ? 0 : begin[e - groups] / block_keys(e); }
  ZB_DEVICE int blocks(int e) const { return (end[e] + block_keys(e) - 1) / block_keys(e) - first_block(e); }
  ZB_DEVICE const int* units_of(int e) const { return units + e + (e < groups ? 0 : 1); }
};

// Which CTAs work on which line: 0 .. of_groups - 1 on that of the groups, the next ones on that of the sequences.  `parts`: into how many pieces a line is cut.
struct Line {
  int parts, total, each, more;  // the first `more` pieces have each + 1 units, the others `each` (at least one)
  ZB_DEVICE void cut(int units, int pieces) {
    total = units;
    parts = min(units, pieces);
    each = parts > 0 ? units / parts : 0;
    more = units - each * parts;
  }
  ZB_DEVICE int first_of(int piece) const { return piece * each + min(piece, more); }
  ZB_DEVICE int owner_of(int unit) const {
    const int split = more * (each + 1);
    return unit < split ? unit / (each + 1) : more + (unit - split) / each;
  }
};
struct Lines {
  int of_groups;
  Line groups, sequences;
};
template <bool SPLIT>
ZB_DEVICE Lines make_lines(int ctas, int of_groups, int of_sequences) {
  Lines l;
  uint32_t a = of_groups, all = of_sequences;
  const int shift = max(0, 12 - __clz(a | all | 1u));      // 20 bits of each
  a = (a >> shift) * (SPLIT ? kTileCost : 1);
  all = a + (all >> shift);
  l.of_groups = of_groups == 0 ? 0 : of_sequences == 0 ? ctas : min(max(static_cast<int>(ctas * (a >> 4) / max(all >> 4, 1u)), 1), ctas - 1);
  l.groups.cut(of_groups, min(l.of_groups, (of_groups + kLeast - 1) / kLeast));
  l.sequences.cut(of_sequences, min((ctas - l.of_groups) * (SPLIT ? kWalkers : 1), SPLIT ? (of_sequences + kLeastSteps - 1) / kLeastSteps : of_sequences));
  return l;
}

struct Segment {                 // the part of an item that a CTA works on
  int entry, tile, head;
  int block, count;              // tiles of 64 keys, from key 64 * block on
};

template <bool SPLIT>
struct Walk {
  int at, to, entry;
  ZB_DEVICE void start(const Plan<SPLIT>& p, int line, int from, int until) {
    at = from;
    to = until;
    int lo = line == 0 ? 0 : p.groups, hi = line == 0 ? p.groups : p.entries;      // the last entry with units <= from
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (*p.units_of(mid) <= from) lo = mid; else hi = mid;
    }
    entry = lo;
  }
  ZB_DEVICE bool next(const Plan<SPLIT>& p, int hkv, Segment& s) {
    while (at < to) {
      while (p.units_of(entry)[1] <= at) ++entry;
      const int n = p.blocks(entry) + kSwitch, local = at - *p.units_of(entry), item = local / n, j = local - item * n, take = min(n - j, to - at);
      at += take;
      s.count = max(j + take - kSwitch, 0) - max(j - kSwitch, 0);
      if (s.count == 0) continue;
      s.entry = entry;
      s.tile = entry < p.groups ? item / hkv : 0;
      s.head = item - s.tile * hkv;
      s.block = max(j - kSwitch, 0) + p.first_block(entry);
      return true;
    }
    return false;
  }
};

ZB_DEVICE void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
ZB_DEVICE void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
ZB_DEVICE void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
ZB_DEVICE void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
ZB_DEVICE void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
ZB_DEVICE uint32_t transpose8(uint32_t x) {          // of 8 x 8 numbers of 16 bits over the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// max of three, one instruction
ZB_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

ZB_DEVICE int clamp_keys(int n, const SharedParams& p) { return min(max(n, 0), p.max_pages * p.page_size); }

// All threads of the CTA.
template <bool SPLIT>
ZB_DEVICE Lines make_plan(const SharedParams& p, Plan<SPLIT>& plan, longlong2* scratch) {
  const int g_n = p.groups, e_n = g_n + p.batch, tid = threadIdx.x;
  for (int i = tid; i < p.listed; i += kThreads) {
    const int b = p.rows[i];
    plan.rows[i] = b >= 0 && b < p.batch ? b : -1;
  }
  for (int g = tid; g <= g_n; g += kThreads) plan.starts[g] = min(max(p.starts[g], 0), p.listed);
  for (int b = tid; b < p.batch; b += kThreads) {
    plan.begin[b] = 0;
    plan.end[g_n + b] = clamp_keys(p.seq_lens[b], p);
  }
  for (int g = tid; g < g_n; g += kThreads) plan.end[g] = clamp_keys(p.lens[g], p);
  __syncthreads();
  // a sequence that is listed twice is where it is listed last: all CTAs have to see it in the same place
  for (int i = tid; i < p.listed; i += kThreads) {
    const int b = plan.rows[i];
    if (b >= 0 && plan.group_of(i) >= 0) atomicMax(&plan.begin[b], i + 1);
  }
  __syncthreads();
  // What a group shares ends with its shortest member, so that every member has every key of a tile: a weight of zero would not make a NaN zero that only longer
  // members see, or nobody.  A member that has ended takes no part, its pages may be anything.
  for (int i = tid; i < p.listed; i += kThreads) {
    const int b = plan.rows[i];
    if (b < 0) continue;
    if (plan.begin[b] != i + 1 || plan.end[g_n + b] == 0) plan.rows[i] = -1;
    else atomicMin(&plan.end[plan.group_of(i)], plan.end[g_n + b]);
  }
  __syncthreads();
  for (int i = tid; i < p.listed; i += kThreads) {
    const int b = plan.rows[i];
    if (b >= 0) plan.begin[b] = plan.end[plan.group_of(i)];
  }
  __syncthreads();
  // sums up to every entry, of both lines: a run of entries a thread, then threads, then warps
  const int each = (e_n + kThreads - 1) / kThreads, e0 = min(tid * each, e_n), e1 = min(e0 + each, e_n);
  const auto count = [&](int e) {
    const int n = plan.blocks(e);
    if (e >= g_n) return plan.end[e] > plan.begin[e - g_n] ? static_cast<long long>(p.hkv) * (n + kSwitch) : 0ll;
    return n > 0 ? static_cast<long long>((max(plan.starts[e + 1] - plan.starts[e], 0) + p.per_tile - 1) / p.per_tile) * p.hkv * (n + kSwitch) : 0ll;
  };
  long long sum[2] = {0, 0};
  for (int e = e0; e < e1; ++e) sum[e >= g_n ? 1 : 0] += count(e);
  long long upto[2] = {sum[0], sum[1]};
  const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long u = __shfl_up_sync(0xffffffffu, upto[i], o);
      if (lane >= o) upto[i] += u;
    }
  if (lane == 31) scratch[warp] = make_longlong2(upto[0], upto[1]);
  __syncthreads();
  long long before[2] = {upto[0] - sum[0], upto[1] - sum[1]}, total[2] = {0, 0};
  for (int w = 0; w < kThreads / 32; ++w) {
    const longlong2 x = scratch[w];
    if (w < warp) before[0] += x.x, before[1] += x.y;
    total[0] += x.x, total[1] += x.y;
  }
  for (int e = e0; e < e1; ++e) {
    const int i = e >= g_n ? 1 : 0;
    plan.units[e + i] = static_cast<int>(before[i]);
    before[i] += count(e);
  }
  if (tid == 0) plan.units[g_n] = static_cast<int>(total[0]), plan.units[e_n + 1] = static_cast<int>(total[1]);
  __syncthreads();
  if (total[0] > 0x3fffffffll || total[1] > 0x3fffffffll) {      // groups that overlap many times over
    if (tid == 0) zb_record_error(p.status, ZB_ERR_BAD_ARG, kKernelId, 20u, static_cast<uint32_t>(total[0] >> 10));
    total[0] = total[1] = 0;
  }
  return make_lines<SPLIT>(gridDim.x, static_cast<int>(total[0]), static_cast<int>(total[1]));
}

// NB: blocks of eight heads of a sequence's own keys that warps 0-3 work on with mma.sync; 0: these go the tensor cores' way, too (more than 16 heads).
template <int HD, int NB>
__global__ void __launch_bounds__(kThreads, Shape<HD>::kCtas)
zb_shared_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_k16,
                        const __grid_constant__ CUtensorMap tmap_v16, const SharedParams p) {
  using S = Shape<HD>;
  constexpr int kStages = S::kStages;
  constexpr bool kSplit = NB > 0;
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
  uint64_t* ring_full = o_ready + 1;                 // [kWalkers][kDepth]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(ring_full + kWalkers * S::kDepth);
  volatile uint32_t* abort_flag = tmem_holder + 1;
  volatile uint32_t* abort_where = tmem_holder + 2;
  Plan<kSplit> plan;
  plan.groups = p.groups;
  plan.entries = p.groups + p.batch;
  plan.starts = reinterpret_cast<int*>(bars + 64);
  plan.end = plan.starts + p.groups + 1;
  plan.begin = plan.end + plan.entries;
  plan.units = plan.begin + p.batch;
  plan.rows = plan.units + plan.entries + 2;
  __shared__ longlong2 scratch[kThreads / 32];

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
    for (int i = 0; i < kWalkers * S::kDepth; ++i) zb_mbar_init(&ring_full[i], 1);
    *abort_flag = 0u;
    *abort_where = 0u;
    zb_mbar_fence_init();
    zb_tma_prefetch_desc(&tmap_k);
    zb_tma_prefetch_desc(&tmap_v);
    if (kSplit) zb_tma_prefetch_desc(&tmap_k16), zb_tma_prefetch_desc(&tmap_v16);
  }
  if (warp == 5) {
    zb_tmem_alloc(tmem_holder, S::kTmemCols);
    zb_tmem_relinquish();
  }
  zb_pdl_wait();                                     // the batch description, queries and keys come from preceding work
  const Lines lines = make_plan<kSplit>(p, plan, scratch);
  zb_tc_fence_before();
  __syncthreads();
  zb_tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  zb_pdl_launch();                                   // only now: a successor that also takes tensor memory must not come first

  // For zb_shared_merge_kernel: where a sequence's parts are.
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < p.batch; b += kThreads) {
      const int e = p.groups + b, *u = plan.units_of(e);
      reinterpret_cast<int4*>(p.where)[2 * b] = make_int4(0, 0, 0, 0);
      reinterpret_cast<int4*>(p.where)[2 * b + 1] = make_int4(lines.sequences.total > 0 && u[1] > u[0] ? plan.blocks(e) : 0, u[0] + kSwitch, lines.groups.total, lines.sequences.total);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.listed; i += kThreads) {
      const int g = plan.group_of(i), b = plan.rows[i];
      if (g < 0 || b < 0 || lines.groups.total == 0 || plan.units[g + 1] == plan.units[g]) continue;
      const int n = plan.blocks(g), at = i - plan.starts[g], tile = at / p.per_tile, first = plan.starts[g] + tile * p.per_tile;
      reinterpret_cast<int4*>(p.where)[2 * b] =
          make_int4(n, plan.units[g] + tile * p.hkv * (n + kSwitch) + kSwitch, first * p.hkv + i - first, min(p.per_tile, plan.starts[g + 1] - first));
    }
  }

  const int line = static_cast<int>(blockIdx.x) < lines.of_groups ? 0 : 1, piece0 = static_cast<int>(blockIdx.x) - (line == 0 ? 0 : lines.of_groups);
  const bool by_warps = kSplit && line == 1;
  Walk<kSplit> walk;
  Segment seg;
  walk.at = walk.to = 0;
  const Line cut = line == 0 ? lines.groups : lines.sequences;
  const auto start = [&](int piece) {
    if (piece < cut.parts) walk.start(plan, line, cut.first_of(piece), cut.first_of(piece + 1));
  };
  if (!by_warps) start(piece0);

  if (by_warps) {
    if constexpr (kSplit) {
      // ------------------------------------------------------------------ keys of single sequences: every warp its own piece of the line
      // S^T = K Q^T (16 keys x 8 heads), O^T += V^T P^T (head_dim x 8 heads), so that few heads waste little.  Steps come through a ring of the warp's own,
      // which it fills itself as it reads, so that no warp waits for another one.
      if (warp < kWalkers) {
        constexpr int kSteps = HD / 16, kDepth = S::kDepth;
        const int walker = piece0 * kWalkers + warp, g = lane >> 2, t = lane & 3;
        uint8_t* ring = smem + warp * kDepth * S::kStepBytes;
        uint64_t* full = ring_full + warp * kDepth;
        start(walker);
        // the loads' way: a lane for each of 32 steps, its first slot of the cache
        Walk<kSplit> l_walk = walk;
        Segment l_seg;
        int l_at = 0, l_slots = 0, l_stage = 0;
        bool l_more = l_walk.next(plan, p.hkv, l_seg);
        const auto slots_of = [&](const Segment& s, int j0) {
          const int key = (s.block + j0 + lane) * kStep;
          if (j0 + lane >= s.count) return -kStep;
          const int page = p.block_table[static_cast<size_t>(s.entry - p.groups) * p.max_pages + key / p.page_size];
          return ZB_BC_OK(page, ZB_BC_PAGES, kKernelId, 2) && page >= 0 ? page * p.page_size + key % p.page_size : -kStep;
        };
        const auto load = [&]() {
          if (!l_more) return;
          if ((l_at & 31) == 0) l_slots = slots_of(l_seg, l_at);
          const int at = __shfl_sync(0xffffffffu, l_slots, l_at & 31);
          if (lane == 0) {
            uint8_t* dst = ring + l_stage * S::kStepBytes;
            zb_mbar_expect_tx(&full[l_stage], S::kStepBytes);
            zb_tma_load_4d(dst, &tmap_k16, &full[l_stage], 0, at, 0, l_seg.head);
            zb_tma_load_4d(dst + S::kStepBytes / 2, &tmap_v16, &full[l_stage], 0, at, 0, l_seg.head);
          }
          if (++l_stage == kDepth) l_stage = 0;
          if (++l_at == l_seg.count) {
            l_at = 0;
            l_more = l_walk.next(plan, p.hkv, l_seg);
          }
        };
#pragma unroll 1
        for (int i = 0; i < kDepth; ++i) load();
        uint32_t stage = 0, phase = 0;
        const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_chunk = lane >> 4;                  // of ldmatrix: a lane's row and piece
        const int v_row = (lane & 7) + (lane >> 4) * 8, v_chunk = (lane >> 3) & 1;
        const auto at = [&](uint32_t tile, int row, int chunk) { return tile + (chunk >> 3) * (kStep * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); };
        bool ok = true;
        while (ok && walk.next(plan, p.hkv, seg)) {
          uint32_t qf[NB][kSteps][2];
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const int head = n * 8 + g;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + (seg.entry - p.groups) * p.q_stride + (seg.head * p.group + head) * HD) + t;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
              qf[n][k][0] = head < p.group ? src[8 * k] : 0u;
              qf[n][k][1] = head < p.group ? src[8 * k + 4] : 0u;
            }
          }
          const int end = plan.end[seg.entry], lo = plan.begin[seg.entry - p.groups];
          float o[NB][kSteps][4], m[NB][2], l[NB][2];
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
          }
          for (int j = 0; j < seg.count; ++j) {
            const int key0 = (seg.block + j) * kStep;
            uint8_t* step = ring + stage * S::kStepBytes;
            const uint32_t kt = zb_smem_u32(step), vt = kt + S::kStepBytes / 2;
            if (!__all_sync(0xffffffffu, zb_mbar_wait(&full[stage], phase, abort_flag))) {
              *abort_where = 16u;
              ok = false;
              break;
            }
            if (key0 + kStep > end) {                // rows of V behind the end hold whatever was there before, perhaps NaN, which a weight of zero does not make zero
              for (int i = lane; i < kStep * S::kSubs * 8; i += 32)
                if (key0 + (i >> 3) % kStep >= end) *reinterpret_cast<uint4*>(step + S::kStepBytes / 2 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
              zb_fence_proxy_async_smem();
              __syncwarp();
            }
            float s[NB][4];
#pragma unroll
            for (int n = 0; n < NB; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
              uint32_t a[4];
              ldmatrix_x4(a, at(kt, k_row, 2 * k + k_chunk));
#pragma unroll
              for (int n = 0; n < NB; ++n) mma_bf16(s[n], a, qf[n][k][0], qf[n][k][1]);
            }
            const bool see0 = key0 + g >= lo && key0 + g < end, see1 = key0 + g + 8 >= lo && key0 + g + 8 < end;
            bool rises = false;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                s[n][i] = (i < 2 ? see0 : see1) ? s[n][i] * p.scale_log2 : -INFINITY;
                rises = rises || s[n][i] > m[n][i & 1] + kLazy;
              }
            }
            if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
              for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float mx = fmaxf(s[n][i], s[n][i + 2]);
                  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                  if (mx > m[n][i]) {
                    const float alpha = m[n][i] == -INFINITY ? 1.f : zb_ex2(m[n][i] - mx);
                    m[n][i] = mx;
                    l[n][i] *= alpha;
#pragma unroll
                    for (int c = 0; c < kSteps; ++c) o[n][c][i] *= alpha, o[n][c][i + 2] *= alpha;
                  }
                }
            }
            uint32_t pb[NB][2];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                s[n][i] = zb_ex2(s[n][i] - (m[n][i & 1] == -INFINITY ? 0.f : m[n][i & 1]));
                l[n][i & 1] += s[n][i];
              }
              pb[n][0] = transpose8(zb_pack_bf16x2(s[n][0], s[n][1]));
              pb[n][1] = transpose8(zb_pack_bf16x2(s[n][2], s[n][3]));
            }
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
              uint32_t a[4];
              ldmatrix_x4_trans(a, at(vt, v_row, 2 * c + v_chunk));
#pragma unroll
              for (int n = 0; n < NB; ++n) mma_bf16(o[n][c], a, pb[n][0], pb[n][1]);
            }
            __syncwarp();                            // the step has been read
            load();
            if (++stage == kDepth) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          const long long to_row = p.own_row + (static_cast<long long>(seg.entry - p.groups) * p.hkv + seg.head + walker) * p.group;
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 4);
              l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 8);
              l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 16);
              const int head = n * 8 + 2 * t + i;
              if (head >= p.group) continue;
              if (g == 0) p.part_ml[to_row + head] = make_float2(m[n][i], l[n][i]);
              float* dst = p.part_o + (to_row + head) * HD + g;
#pragma unroll
              for (int c = 0; c < kSteps; ++c) {
                dst[c * 16] = o[n][c][i];
                dst[c * 16 + 8] = o[n][c][i + 2];
              }
            }
        }
      }
    }
  } else if (warp == 4) {
    // ------------------------------------------------------------------ TMA producer
    // Pages of 64 tokens and more come as one box of all columns; of smaller ones several make up a tile, a box each and 64 columns.
    const int box = min(p.page_size, kKeys), pages_of_tile = kKeys / box, at_once = 32 / pages_of_tile;
    // A lane for each box of tiles j0 .. j0 + at_once - 1 of an item's part: its first slot of the cache.  Behind the end it lies outside of the cache, which
    // reads as zeros.
    const auto slots_of = [&](const Segment& g, int j0) {
      int seq = 0;
      if (g.entry >= p.groups) {
        seq = g.entry - p.groups;
      } else {                                       // any member's pages are the group's
        for (int i = plan.starts[g.entry]; i < plan.starts[g.entry + 1]; ++i) {
          if (plan.rows[i] < 0) continue;
          seq = plan.rows[i];
          break;
        }
      }
      const int key = (g.block + j0) * kKeys + lane * box;
      if (key >= plan.end[g.entry] || j0 + lane / pages_of_tile >= g.count) return -kKeys;
      const int page = p.block_table[static_cast<size_t>(seq) * p.max_pages + key / p.page_size];
      return ZB_BC_OK(page, ZB_BC_PAGES, kKernelId, 1) && page >= 0 ? page * p.page_size + key % p.page_size : -kKeys;
    };
    // A tile of K (w = 0) or V, number t of the walk, whose slots the lanes hold.
    const auto load = [&](int w, int t, int slot, int head) {
      const int stage = t % kStages;
      uint64_t *full = (w == 0 ? k_full : v_full) + stage, *empty = (w == 0 ? k_empty : v_empty) + stage;
      if (t >= kStages && !__all_sync(0xffffffffu, zb_mbar_wait(empty, static_cast<uint32_t>(t / kStages - 1) & 1u, abort_flag))) {
        *abort_where = 1u;
        return false;
      }
      uint8_t* dst = (w == 0 ? k_s : v_s) + stage * S::kKvBytes;
      const CUtensorMap* map = w == 0 ? &tmap_k : &tmap_v;
      if (lane == 0) zb_mbar_expect_tx(full, S::kKvBytes);
      __syncwarp();
      if (pages_of_tile == 1) {
        if (lane == 0) zb_tma_load_4d(dst, map, full, 0, slot, 0, head);
      } else if (lane < pages_of_tile) {
#pragma unroll
        for (int c = 0; c < S::kSubs; ++c) zb_tma_load_4d(dst + c * (kKeys * 128) + lane * box * 128, map, full, 0, slot, c, head);
      }
      return true;
    };
    int done = 0, slots = 0, v_slot = 0, v_head = 0;
    bool ok = true, more = walk.next(plan, p.hkv, seg);
    if (more) slots = slots_of(seg, 0);
    while (ok && more) {
      Segment next;
      int next_slots = 0;
      more = walk.next(plan, p.hkv, next);
      if (more) next_slots = slots_of(next, 0);      // asked for an item ahead
      for (int j = 0; ok && j < seg.count; ++j, ++done) {
        if (j > 0 && j % at_once == 0) slots = slots_of(seg, j);
        const int slot = __shfl_sync(0xffffffffu, slots, (j % at_once * pages_of_tile + lane) & 31);
        // K a tile ahead of V: its room is free as soon as S is done
        ok = load(0, done, slot, seg.head) && (done == 0 || load(1, done - 1, v_slot, v_head));
        v_slot = slot;
        v_head = seg.head;
      }
      seg = next;
      slots = next_slots;
    }
    if (ok && done > 0) load(1, done - 1, v_slot, v_head);
  } else if (warp == 5) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t kIdescS = zb_make_idesc_bf16(kRows, kKeys);
      constexpr uint32_t kIdescO = zb_make_idesc_bf16(kRows, HD) | (1u << 16);         // B (= V) is MN-major
      const uint32_t t_s = tmem_base, t_o = tmem_base + S::kColO, qa = zb_smem_u32(q_s);
      uint32_t k_stage = 0, k_phase = 0, stage = 0, phase = 0, where = 0;
      int s_done = 0, done = 0, segment = 0, ahead = 0;
      Walk<kSplit> s_walk = walk;
      Segment s_seg;
      // S of the next tile, whatever item it is of, into the buffer that is its number's parity.  Behind an item's last S the softmax warps bring in the next item's
      // queries, while that S is worked on.
      const auto next_s = [&]() {
        if (ahead == 0) {
          if (!s_walk.next(plan, p.hkv, s_seg)) return true;
          ahead = s_seg.count;
          if (!zb_mbar_wait(q_full, static_cast<uint32_t>(segment) & 1u, abort_flag)) {
            where = 2u;
            return false;
          }
          ++segment;
        }
        --ahead;
        if (!zb_mbar_wait(&k_full[k_stage], k_phase, abort_flag)) {
          where = 3u;
          return false;
        }
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
      bool ok = next_s() && next_s();
      while (ok && walk.next(plan, p.hkv, seg)) {
        for (int j = 0; ok && j < seg.count; ++j) {
          if (!zb_mbar_wait(&v_full[stage], phase, abort_flag)) {
            where = 4u;
            ok = false;
            break;
          }
          if (!zb_mbar_wait(&p_full[done & 1], static_cast<uint32_t>(done >> 1) & 1u, abort_flag)) {
            where = 5u;
            ok = false;
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
          ++done;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
          ok = next_s();                             // over P, in order behind the MMAs that read it
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
    constexpr int kPieces = HD / 8, kAhead = HD / 64;     // 16-byte pieces of a row; of the next item's queries, those that a thread asks for ahead
    struct Item {
      int first, seqs, rows, end, lo;
      bool common;
    };
    const auto item_of = [&](const Segment& g) {     // row i of an item is head i % group of its sequence i / group
      Item i;
      i.common = g.entry < p.groups;
      i.first = i.common ? plan.starts[g.entry] + g.tile * p.per_tile : 0;
      i.seqs = i.common ? min(p.per_tile, plan.starts[g.entry + 1] - i.first) : 1;
      i.rows = i.seqs * p.group;
      i.end = plan.end[g.entry];
      i.lo = i.common ? 0 : plan.begin[g.entry - p.groups];
      return i;
    };
    const uint32_t inverse = (65536u + p.group - 1) / p.group;      // row / group of up to 128 rows is row * inverse >> 16
    const auto sequence_of = [&](const Segment& g, const Item& i, int nth) { return i.common ? plan.rows[i.first + nth] : g.entry - p.groups; };
    const auto piece_at = [&](const Segment& g, const Item& i, int n) {
      const int row = n / kPieces, nth = row * inverse >> 16, seq = max(sequence_of(g, i, nth), 0);
      return reinterpret_cast<const uint4*>(p.q + seq * p.q_stride + (g.head * p.group + row - nth * p.group) * HD + n % kPieces * 8);
    };
    const auto room_of = [&](int n) {
      const int row = n / kPieces, piece = n % kPieces;
      return q_s + (piece >> 3) * (kRows * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
    };
    const auto copy_queries = [&](const Segment& g, const Item& i) {      // all on their way together
#pragma unroll 4
      for (int n = threadIdx.x; n < i.rows * kPieces; n += kRows) copy16(zb_smem_u32(room_of(n)), piece_at(g, i, n));
      copies_done();
    };
    const auto publish_queries = [&]() {
      zb_fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) zb_mbar_arrive(q_full);
    };
    int it = 0;                                      // tiles so far
    bool ok = true, more = walk.next(plan, p.hkv, seg);
    Item item;
    if (more) {
      item = item_of(seg);
      copy_queries(seg, item);
      publish_queries();
    }
    float* owed = nullptr;                           // where the item before goes, once its O is complete
    bool owes = false;
    const auto settle = [&]() {                      // O of the item before, up to tile it - 1
      if (!__all_sync(0xffffffffu, zb_mbar_wait(o_ready, static_cast<uint32_t>(it - 1) & 1u, abort_flag))) {
        *abort_where = 14u;
        return false;
      }
      if (__any_sync(0xffffffffu, owed != nullptr)) {
        zb_tc_fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += 32) {
          uint32_t o[32];
          zb_tmem_ld32(t_o + c0, o);
          zb_tmem_ld_wait();
          if (owed != nullptr) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(owed + c0 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      owes = false;
      return true;
    };
    while (ok && more) {
      Segment next;
      Item after;
      more = walk.next(plan, p.hkv, next);
      uint4 piece[kAhead];
      int pieces = 0;
      if (more) {
        after = item_of(next);
        pieces = after.rows * kPieces;
        if (pieces <= kAhead * kRows) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
            if (threadIdx.x + i * kRows < pieces) piece[i] = *piece_at(next, after, threadIdx.x + i * kRows);
        }
      }
      const int end = item.end, lo = item.lo;
      const bool mine = warp * 32 < item.rows, row_valid = r < item.rows;
      const int limit = item.common && row_valid && sequence_of(seg, item, r * inverse >> 16) < 0 ? 0 : end;      // (a row of no sequence sees nothing)
      const int least = __reduce_min_sync(0xffffffffu, limit);
      float m = -INFINITY, l = 0.f;
      bool whole = false;                            // some row's reference is so large that fp32 has whole numbers only
      for (int j = 0; j < seg.count; ++j, ++it) {
        const int b = it & 1;
        const uint32_t t_s = tmem_base + b * kKeys + lane_off;
        if (!__all_sync(0xffffffffu, zb_mbar_wait(&s_full[b], static_cast<uint32_t>(it >> 1) & 1u, abort_flag))) {
          *abort_where = 10u;
          ok = false;
          break;
        }
        zb_tc_fence_after();
        if (more && j == seg.count - 1) {            // the queries have been read for the last time
          if (pieces <= kAhead * kRows) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
              if (threadIdx.x + i * kRows < pieces) *reinterpret_cast<uint4*>(room_of(threadIdx.x + i * kRows)) = piece[i];
          } else {
            copy_queries(next, after);
          }
          publish_queries();
        }
        const int key0 = (seg.block + j) * kKeys;
        if (mine) {
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
          const bool moves = mx > m + kLazy && row_valid;      // also the first visible key: m = -inf
          if (moves) {
            alpha = m == -INFINITY ? 1.f : zb_ex2(m - mx);
            m = mx;
            l *= alpha;
          }
          const bool some_move = __any_sync(0xffffffffu, moves);
          if (some_move) whole = __any_sync(0xffffffffu, fabsf(m) > 0x1p24f && m != -INFINITY);
          if (some_move && j > 0) {
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
          ZbF2 sum[2] = {0ull, 0ull};
          if (whole) {                               // products rounded as m is: of others the largest one's is off by half a step of m, 2^7 from 2^31 on
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t x[32];
              zb_tmem_ld32(t_s + 32 * c, x);
              zb_tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float e[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const int key = key0 + 32 * c + i + k;
                  e[k] = key < limit && key >= lo ? zb_ex2(__fadd_rn(__fmul_rn(__uint_as_float(x[i + k]), p.scale_log2), neg_m)) : 0.f;
                }
                sum[0] = zb_add2(sum[0], zb_pack2(e[0], e[1]));
                x[i / 2] = zb_pack_bf16x2(e[0], e[1]);
              }
              zb_tmem_st16(t_s + 16 * c, x);         // (what these columns held has been read)
            }
          } else {
            const ZbF2 nm2 = zb_pack2(neg_m, neg_m);
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
        // The item before still has its O where this one's goes.
        if (owes && !settle()) {
          ok = false;
          break;
        }
        // Parity does not tell a phase of o_ready from the one two before it, so that no wait may begin two phases early: S of a tile went behind P V of the
        // tile two in front, but at the end no further S tells, and the last tile but one is waited for while the last one is held back.
        if (!more && j > 0 && j == seg.count - 1 && !__all_sync(0xffffffffu, zb_mbar_wait(o_ready, static_cast<uint32_t>(it - 1) & 1u, abort_flag))) {
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
      owed = nullptr;
      owes = true;
      if (row_valid) {
        // rows of parts, disjoint: an item's own, and as many again for every CTA in front
        const long long at = (item.common ? (static_cast<long long>(item.first) * p.hkv + seg.head * item.seqs) * p.group + static_cast<long long>(piece0) * kRows
                                          : p.own_row + (static_cast<long long>(seg.entry - p.groups) * p.hkv + seg.head + piece0) * p.group) + r;
        p.part_ml[at] = make_float2(m, l);
        owed = p.part_o + at * HD;
      }
      seg = next;
      item = after;
    }
    if (ok && owes) settle();
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

// The rows of one (sequence, key head), over all parts that the kernel above left of them.  where[seq] = {blocks of the prefix, first unit of them (of key head
// 0), row of its parts in units of `group` (likewise), step of these to the next key head; blocks of its own, first unit of them, units of both lines}.  A warp
// works on a row, or 2, 4, .. 16 on one: what bounds the kernel is the chain of loads, not their number (8 sequences of
// 34 parts, a warp a row: 9 us; four: 18.8 us for the whole call, 16: 17.7).
template <int HD, bool SPLIT>
__global__ void __launch_bounds__(512)
zb_shared_merge_kernel(const int32_t* __restrict__ where, const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                       __nv_bfloat16* __restrict__ out, int hkv, int group, int log2_warps, int own_row, int part_rows, int ctas) {
  constexpr int kEach = HD / 32, kOnce = HD == 256 ? 4 : 8;      // parts that are on their way together
  __shared__ float sums[16][HD];
  __shared__ float2 stats[16];
  zb_pdl_launch();
  zb_pdl_wait();
  const int b = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 front = reinterpret_cast<const int4*>(where)[2 * b], back = reinterpret_cast<const int4*>(where)[2 * b + 1];
  const Lines lines = make_lines<SPLIT>(ctas, back.z, back.w);
  int n0 = 0, n1 = 0, c0 = 0, c1 = 0;
  if (front.x > 0) {
    const int u = front.y + head * (front.x + kSwitch);
    c0 = lines.groups.owner_of(u);
    n0 = lines.groups.owner_of(u + front.x - 1) - c0 + 1;
  }
  if (back.x > 0) {
    const int u = back.y + head * (back.x + kSwitch);
    c1 = lines.sequences.owner_of(u);
    n1 = lines.sequences.owner_of(u + back.x - 1) - c1 + 1;
  }
  const int n = n0 + n1, warps = 1 << log2_warps, share = warp & (warps - 1);
  const int r = blockIdx.z * (16 >> log2_warps) + (warp >> log2_warps);
  float acc[kEach], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < kEach; ++j) acc[j] = 0.f;
  if (r < group) {
    const long long row0 = (static_cast<long long>(front.z) + static_cast<long long>(head) * front.w) * group + static_cast<long long>(c0) * kRows + r;
    const long long row1 = own_row + (static_cast<long long>(b) * hkv + head + c1) * group + r;
    const auto place = [&](int i) {                // (a sequence that is in two groups finds a wrong row, but one that is there)
      const long long at = i < n0 ? row0 + static_cast<long long>(i) * kRows : row1 + static_cast<long long>(i - n0) * group;
      return at < part_rows ? at : 0ll;
    };
    const int mine = (n - share + warps - 1) >> log2_warps;      // parts share, share + warps, ..
    for (int i0 = 0; i0 < mine; i0 += kOnce) {
      float x[kOnce][kEach];
      float2 ml = make_float2(-INFINITY, 0.f);
      if (lane < kOnce && i0 + lane < mine) ml = part_ml[place(share + ((i0 + lane) << log2_warps))];
#pragma unroll
      for (int i = 0; i < kOnce; ++i) {
        const float2* src = reinterpret_cast<const float2*>(part_o + place(share + (min(i0 + i, mine - 1) << log2_warps)) * HD + lane * kEach);
#pragma unroll
        for (int j = 0; j < kEach / 2; ++j) {
          const float2 y = src[j];
          x[i][2 * j] = y.x, x[i][2 * j + 1] = y.y;
        }
      }
      const float up = fmaxf(top, zb_warp_max(ml.x)), base = up == -INFINITY ? 0.f : up;
      const float was = zb_ex2(top - base), f = zb_ex2(ml.x - base);
      top = up;
      sum = sum * was + zb_warp_sum(f * ml.y);
#pragma unroll
      for (int j = 0; j < kEach; ++j) acc[j] *= was;
#pragma unroll
      for (int i = 0; i < kOnce; ++i) {
        if (i0 + i >= mine) break;
        const float by = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
        for (int j = 0; j < kEach; ++j) acc[j] += by * x[i][j];
      }
    }
  }
  if (warps > 1) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) sums[warp][lane * kEach + j] = acc[j];
    if (lane == 0) stats[warp] = make_float2(top, sum);
    __syncthreads();
    if (share == 0 && r < group) {
      float most = top;
      for (int w = 1; w < warps; ++w) most = fmaxf(most, stats[warp + w].x);
      const float base = most == -INFINITY ? 0.f : most, f = zb_ex2(top - base);
      sum *= f;
#pragma unroll
      for (int j = 0; j < kEach; ++j) acc[j] *= f;
      for (int w = 1; w < warps; ++w) {
        const float g = zb_ex2(stats[warp + w].x - base);
        sum += g * stats[warp + w].y;
#pragma unroll
        for (int j = 0; j < kEach; ++j) acc[j] += g * sums[warp + w][lane * kEach + j];
      }
    }
  }
  if (share == 0 && r < group) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;      // no key at all: zeros
    __nv_bfloat16* dst = out + (static_cast<size_t>(b) * hkv * group + head * group + r) * HD + lane * kEach;
#pragma unroll
    for (int j = 0; j < kEach; j += 2) *reinterpret_cast<uint32_t*>(dst + j) = zb_pack_bf16x2(acc[j] * inv, acc[j + 1] * inv);
  }
}

int plan_bytes(int batch, int groups) { return 4 * (groups + 1 + (groups + batch) + batch + groups + batch + 2 + batch); }

// CTAs of the walk: as many as fit at once.
template <int HD>
int walk_ctas(int batch, int groups, int sms) {
  const int smem = Shape<HD>::kSmem + plan_bytes(batch, groups);
  return sms * (Shape<HD>::kCtas == 2 && 2 * (smem + 1024) <= 228 * 1024 ? 2 : 1);
}
int walk_ctas(int hd, int batch, int groups, int sms) {
  return hd == 64 ? walk_ctas<64>(batch, groups, sms) : hd == 128 ? walk_ctas<128>(batch, groups, sms) : walk_ctas<256>(batch, groups, sms);
}

// Blocks of eight heads that single warps take of sequences' own keys; 0: these are tiles, too.
int own_blocks(int group) { return group <= 8 ? 1 : group <= 16 ? 2 : 0; }

// Rows of the parts: of prefixes (from row 0 on) and of the sequences' own keys, whose line is cut into pieces for warps or, as tiles, for CTAs.
long long prefix_rows(int listed, int hq, int ctas) { return static_cast<long long>(listed) * hq + static_cast<long long>(ctas) * kRows; }
long long part_rows(int listed, int batch, int hq, int group, int ctas) {
  const int pieces = ctas * (own_blocks(group) > 0 ? kWalkers : 1);
  return (prefix_rows(listed, hq, ctas) + static_cast<long long>(batch) * hq + static_cast<long long>(pieces) * group + 1) & ~1ll;      // (16 bytes)
}

template <int HD, int NB>
int launch(const CUtensorMap (&maps)[4], const SharedParams& p, void* out, int rows, int ctas, cudaStream_t s) {
  static bool configured[16] = {};
  if (const int rc = zb_config_smem_once(zb_shared_decode_kernel<HD, NB>, Shape<HD>::kSmem + plan_bytes(kMaxBatch, kMaxBatch), configured)) return rc;
  cudaError_t e = zb_launch(zb_shared_decode_kernel<HD, NB>, dim3(ctas), dim3(kThreads), Shape<HD>::kSmem + plan_bytes(p.batch, p.groups), s, maps[0], maps[1], maps[2], maps[3], p);
  // as many warps a row as a CTA for a head's rows has; more where there are few rows
  int log2_warps = p.group > 8 ? 0 : p.group > 4 ? 1 : p.group > 2 ? 2 : p.group == 2 ? 3 : 4;
  const auto merge_ctas = [&](int log2) { return static_cast<long long>(p.batch) * p.hkv * ((p.group + (16 >> log2) - 1) / (16 >> log2)); };
  while (log2_warps < 4 && merge_ctas(log2_warps + 1) <= 2 * zb_num_sms()) ++log2_warps;
  if (e == cudaSuccess)
    e = zb_launch(zb_shared_merge_kernel<HD, (NB > 0)>, dim3(p.batch, p.hkv, (p.group + (16 >> log2_warps) - 1) / (16 >> log2_warps)), dim3(512), 0, s, p.where, p.part_o,
                  p.part_ml, reinterpret_cast<__nv_bfloat16*>(out), p.hkv, p.group, log2_warps, p.own_row, rows, ctas);
  zb_count_launch(2);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}
template <int HD>
int launch(const CUtensorMap (&maps)[4], const SharedParams& p, void* out, int rows, int ctas, cudaStream_t s) {
  switch (own_blocks(p.group)) {
    case 1: return launch<HD, 1>(maps, p, out, rows, ctas, s);
    case 2: return launch<HD, 2>(maps, p, out, rows, ctas, s);
    default: return launch<HD, 0>(maps, p, out, rows, ctas, s);
  }
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
  CUtensorMap maps[4];                               // tiles of K and V, steps of K and V
  for (int i = 0; i < 4; ++i) {
    const void* cache = i % 2 == 0 ? c->k_cache : c->v_cache;
    const int rc = i < 2 ? zb_make_tmap_kv_box(&maps[i], cache, slots, c->hkv, c->hd, box, subs) : zb_make_tmap_kv_box(&maps[i], cache, slots, c->hkv, c->hd, kStep, c->hd / 64);
    if (rc != 0) return rc;
  }
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
  if (c->hd == 64) return launch<64>(maps, p, c->out, n, ctas, s);
  return c->hd == 128 ? launch<128>(maps, p, c->out, n, ctas, s) : launch<256>(maps, p, c->out, n, ctas, s);
}

}  // extern "C"
