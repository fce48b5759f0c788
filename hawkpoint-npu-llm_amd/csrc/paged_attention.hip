// Attention of a batch's new tokens over a paged KV cache (hk_paged_attention).
//
// Row (token t of an entry, head h) stands at position p = length - count + t
// and sees the slots j <= p (with a window, j > p - window) whose page exists:
//   s_j = scale (q . k_j),  m = max s_j,  l = sum exp(s_j - m)
//   out = sum exp(s_j - m) v_j / l,  lse = m + ln l
// in one pass over the slots with a running maximum and sum.  The rows of all
// query heads of a kv head are rows of the same tiles, and a tile reads K and V
// once for all its rows (16, 32 or 128 of them).  S^T = K Q^T puts a row's
// scores into the lanes that hold the row's column of P^T, the right operand of
// O^T = V^T P^T: the probabilities never leave their registers.  They are
// rounded to bf16 there, 2^-8 of each at most, about what the rounding of the
// result costs: the results are off from float64 by 0.0017 to 0.0020 of their
// norm, where float32 probabilities, rounded once at the end, are off by 0.0016
// to 0.0017 (the prefill kernel's split into three bf16 terms would triple the
// products).  Scores, maxima and sums are float32, and the sum is that of the
// probabilities before their rounding, or lse would be off by 4e-4.
//
// The work of a batch is cut into equal runs of blocks (paged_plan.h), which
// every workgroup works out by itself from the lengths on the device: a batch
// of mixed lengths fills the GPU, a captured launch fits every later length,
// and there is nothing to plan between the calls.  A task that is cut leaves
// (max, sum, O) of its parts in the workspace, and the workgroup that arrives
// last (a ticket per task, zero between launches) joins them in their order.
#include <type_traits>

#include "hk_common.h"
#include "hk_internal.h"
#include "paged.h"
#include "paged_plan.h"

namespace hk {
namespace {

typedef short v4s16 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// buffer access cache policies
constexpr int kSc1 = 16;    // device scope
constexpr int kStream = 2;  // read once: does not stay in the caches
constexpr int kNowhere = 0x7ffffff0;  // an offset past any resource: reads zero, no memory access

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The load of v is waited for here.
__device__ __forceinline__ void settle(bf16x8& v) {
#if __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(v));
#endif
}

// A table entry at a uniform place, through the scalar cache: a vector load
// would be waited for together with the K and V loads in flight.
__device__ __forceinline__ int table_at(const int32_t* table, int i) {
  return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)table)[i];
}

// ---- a workgroup's run of the work ----

// What a task costs beside its blocks: its first loads' latency, its end and,
// for a cut one, the workspace, in halves of a block.  Without it the
// workgroups that have many short tasks end last (190 chats: 69 us against 64,
// pieces of prompts beside chats 72 and 62; one half more or less is the same).
constexpr int kBlockCost = 2, kNarrowTaskCost = 3, kWideTaskCost = 3;

struct Entry {
  int seq, row0;  // sequence (-1: none), first row
  PlanEntry e;
};
// Entry b (uniform), through the scalar cache: entry_rows and entry_seq.
__device__ __forceinline__ Entry load_entry(const PagedAttnArgs& a, int b) {
  const int f0 = min(max(table_at(a.b.first, b), 0), a.b.tokens);
  const int f1 = min(max(table_at(a.b.first, b + 1), f0), a.b.tokens);
  const int s = a.b.seqs ? table_at(a.b.seqs, b) : b;
  const bool is = (unsigned)s < (unsigned)a.c.seqs;
  const int length = is ? min(max(table_at(a.c.length, s), 0), a.c.width << a.c.page_shift) : 0;
  return {is ? s : -1, f0, {length, f1 - f0}};
}

// Whether an entry of `count` rows is this form's (a batch may have long and
// short entries).
__device__ __forceinline__ bool takes(const PagedAttnArgs& a, int count) {
  return count > 0 && count * a.group >= a.rows_min && count * a.group <= a.rows_max;
}

// v of another lane as the DPP control says; 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
// Sum of v over the lanes up to this one: within rows of 16, then the rows
// before.  (With these and without barriers for up to 64 entries 16 chats' check
// of five tokens takes 20.0 us; with __shfl_up through the LDS crossbar and the
// workgroup's barriers it took 21.0.)
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
  v += dpp<0x111, 0xf>(v);  // row_shr:1
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);  // row_bcast:15, to rows 1 and 3
  v += dpp<0x143, 0xc>(v);  // row_bcast:31, to rows 2 and 3
  return v;
}
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
  return (int64_t)((uint64_t)(uint32_t)lane_of((int)(v >> 32), lane) << 32 | (uint32_t)lane_of((int)v, lane));
}

// Sum of v over the workgroup in every thread, and the sum of the threads
// before this one.
__device__ __forceinline__ int64_t scan(int64_t v, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t s = wave_scan(v);
  __syncthreads();
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  return before + s - v;
}

// plan_head_units and plan_find (paged_plan.h), a wave's lanes taking 64 tiles
// at a time: one thread that walked the tiles of a prompt's piece took 12 us
// for 701 tokens and 32 us for 2039.  The arguments are uniform.
__device__ __forceinline__ int64_t wave_units(const PlanShape& s, const PlanEntry& e, int tile) {
  return tile < plan_tiles(s, e) ? plan_units(s, plan_span(s, e, tile)) : 0;
}
__device__ __forceinline__ int64_t wave_head_units(const PlanShape& s, const PlanEntry& e) {
  int64_t n = 0;
  const int tiles = plan_tiles(s, e);
  for (int t = threadIdx.x & 63; t < tiles; t += 64) n += plan_units(s, plan_span(s, e, t));
  return lane_of(wave_scan(n), 63);
}
__device__ __forceinline__ PlanPlace wave_find(const PlanShape& s, const PlanEntry& e, int entry, int64_t start, int64_t rem) {
  const int lane = threadIdx.x & 63, tiles = plan_tiles(s, e);
  const int64_t per_head = tiles == 1 ? plan_units(s, plan_span(s, e, 0)) : wave_head_units(s, e);
  PlanPlace p = {entry, uniform((int)plan_div(rem, per_head)), 0, 0};
  rem -= p.head * per_head;
  start += p.head * per_head;
  p.start = start;
  if (tiles == 1) return p;
  for (;; p.tile += 64) {
    const int64_t u = wave_units(s, e, p.tile + lane);
    const int64_t sum = wave_scan(u);
    const unsigned long long past = __ballot(sum > rem);
    if (past == 0 && p.tile + 64 < tiles) {
      const int64_t all = lane_of(sum, 63);
      rem -= all;
      p.start += all;
      continue;
    }
    const int at = past ? __builtin_ctzll(past) : 63;
    p.tile += at;
    p.start += lane_of(sum - u, at);
    return p;
  }
}

struct Run {
  PlanRun r;
  PlanPlace place;
  Entry entry;
  PlanEven even;  // splits > 0: parts of equal length instead of runs
  int task;       // of those, the workgroup's next task
};

// This workgroup's run; false: it has none.
template <bool EVEN>
__device__ __forceinline__ bool plan_run(const PagedAttnArgs& a, const PlanShape& s, int least, Run& run) {
  __shared__ int64_t sums[kWaves];
  __shared__ int64_t found_start;
  __shared__ int found[5];
  const int n = a.b.n;
  run.even = {0, 0};
  auto cut = [&](int64_t total) { return plan_cut(s, total, gridDim.x, least, blockIdx.x, run.r); };
  if (n == 1) {  // nothing to add up: no barrier
    run.entry = load_entry(a, 0);
    if (!takes(a, run.entry.e.count)) return false;
    const int64_t head = plan_tiles(s, run.entry.e) == 1 ? plan_units(s, plan_span(s, run.entry.e, 0)) : wave_head_units(s, run.entry.e);
    if constexpr (EVEN) {
      run.even = plan_even(s, run.entry.e, s.heads * head, gridDim.x);
      if (run.even.splits) {
        run.r.w = plan_even_number(blockIdx.x, gridDim.x);
        run.task = run.r.w / run.even.splits;
        return run.task < run.even.tasks;
      }
    }
    if (!cut(s.heads * head)) return false;
    run.place = wave_find(s, run.entry.e, 0, 0, run.r.begin);
    return true;
  }
  int2 rows, seq;
  auto units = [&](int b) -> int64_t {
    rows = seq = make_int2(0, 0);
    if (b < n) {
      rows = entry_rows(a.b, b);
      seq = entry_seq(a.c, a.b, b);
    }
    const PlanEntry e = {seq.y, rows.y - rows.x};
    const bool has = b < n && takes(a, e.count), few = has && e.count * s.group <= 4 * s.rows;
    int64_t u = few ? s.heads * plan_head_units(s, e) : 0;
    // entries of more tiles: the wave's lanes together
    for (unsigned long long todo = __ballot(has && !few); todo; todo &= todo - 1) {
      const int l = __builtin_ctzll(todo);
      const int64_t v = wave_head_units(s, {lane_of(e.length, l), lane_of(e.count, l)});
      if ((int)(threadIdx.x & 63) == l) u = s.heads * v;
    }
    return u;
  };
  if (n <= 64) {  // each wave knows all entries: no barrier
    const int64_t mine = units(threadIdx.x & 63), sum = wave_scan(mine);
    if (!cut(lane_of(sum, 63))) return false;
    const int64_t before = sum - mine;
    const int l = __builtin_ctzll(__ballot(before <= run.r.begin && run.r.begin < sum));
    run.entry = {lane_of(seq.x, l), lane_of(rows.x, l), {lane_of(seq.y, l), lane_of(rows.y - rows.x, l)}};
    run.place = wave_find(s, run.entry.e, l, lane_of(before, l), run.r.begin - lane_of(before, l));
    return true;
  }
  // (up to as many entries as threads, the units are worked out once)
  int64_t mine = units(threadIdx.x), total, before = scan(mine, sums, total);
  if (n > kThreads) {
    int64_t all = total;
    for (int b0 = kThreads; b0 < n; b0 += kThreads) {
      scan(units(b0 + threadIdx.x), sums, total);
      all += total;
    }
    total = all;
  }
  total = uniform(total);
  if (!cut(total)) return false;
  int64_t base = 0;
  for (int b0 = 0; b0 < n; b0 += kThreads) {
    int64_t chunk = 0;
    if (b0 > 0) {
      mine = units(b0 + threadIdx.x);
      before = base + scan(mine, sums, chunk);
    } else if (n > kThreads) {
      mine = units(threadIdx.x);
      scan(mine, sums, chunk);
    }
    if (before <= run.r.begin && run.r.begin < before + mine) {
      found[0] = b0 + threadIdx.x;
      found[1] = seq.x, found[2] = rows.x, found[3] = seq.y, found[4] = rows.y - rows.x;
      found_start = before;
    }
    base += chunk;
  }
  __syncthreads();
  const int b = uniform(found[0]);
  const int64_t start = uniform(found_start);
  run.entry = {uniform(found[1]), uniform(found[2]), {uniform(found[3]), uniform(found[4])}};
  run.place = wave_find(s, run.entry.e, b, start, run.r.begin - start);
  return true;
}

// A workgroup's part of a task: blocks [kb0, kb1) of the `rows` rows from r0 of
// kv head g, of which it sees slots below `seen`.
struct Task {
  Entry entry;
  const int32_t* table;  // the sequence's pages
  int g, tile, r0, rows, pos0, kb0, kb1, seen;
  bool cut;
  PlanParts parts;  // of a cut task
};

// Fills in t for the workgroup's part of a task.
__device__ __forceinline__ void set_task(const PagedAttnArgs& a, const PlanShape& s, const Entry& entry, const PlanTask& p,
                                         Task& t) {
  t.entry = entry;
  t.table = a.c.table + (int64_t)max(entry.seq, 0) * a.c.width;
  t.g = p.head;
  t.tile = p.tile;
  t.r0 = p.tile * s.rows;
  t.rows = min(s.rows, entry.e.count * a.group - t.r0);
  t.pos0 = entry.e.length - entry.e.count;
  t.kb0 = p.span.lo + p.mine.first;
  t.kb1 = p.span.hi > p.span.lo ? p.span.lo + p.mine.end : t.kb0;
  t.seen = p.span.seen;
  t.cut = p.cut;
  t.parts = p.parts;
}

// The workgroup's next part of a task; false: there is none.
template <bool EVEN>
__device__ __forceinline__ bool next_task(const PagedAttnArgs& a, const PlanShape& s, Run& run, Task& t) {
  if (EVEN && run.even.splits) {
    PlanTask p;
    if (!plan_even_take(s, run.entry.e, run.even, run.r.w, gridDim.x, run.task, p)) return false;
    set_task(a, s, run.entry, p, t);
    return true;
  }
  return plan_take(
      s, run.r, run.entry.e, run.place, [&](const PlanTask& p) { set_task(a, s, run.entry, p, t); },
      [&](PlanPlace& p) {
        while (++p.entry < a.b.n) {
          run.entry = load_entry(a, p.entry);
          if (takes(a, run.entry.e.count)) return;
        }
      });
}

// 2^(score - max): where all scores are -inf the maximum is no number to subtract.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

// What a product q . k is multiplied by, for powers of two.  Not zero where
// tiny factors underflow: a hidden score is -inf times it.  Not an infinity
// where large ones overflow: a product of 0 is a score of 0.
template <bool E4M3>
__device__ __forceinline__ float score_scale(const PagedAttnArgs& a, int g) {
  const float s = (E4M3 ? a.c.k_scale[g] : 1.0f) * a.scale * kLog2e;
  return fminf(fmaxf(s, __builtin_bit_cast(float, 1u)), __FLT_MAX__);
}

// Whether one of the eight bf16 values is an infinity or NaN.
__device__ __forceinline__ bool not_finite(const u32x4& v) {
  bool bad = false;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    bad |= (v[w] & 0x7f80u) == 0x7f80u || (v[w] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// Four e4m3 values as two bf16 pairs (exact: every e4m3 value is a bf16 value;
// v_cvt_scalef32_pk_bf16_fp8 with scale 1).
__device__ __forceinline__ u32x2_t e4m3_bf16(uint32_t w) {
  return u32x2_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
}

// ---- cut tasks ----

// A task whose result is one of several parts: where it starts in the order of
// units, and what is written when all parts are there.
struct Pending {
  PlanParts parts;
  Entry entry;
  int head, tile;
};

// Once the workgroup's parts are stored: draws the tickets of its (at most
// two) cut tasks, and says which of them it has to join, as bits.  The stores
// have completed before the tickets are drawn (device-coherent stores, no L2
// write-back as a fence would do).  The joining workgroup leaves the ticket at
// zero.
__device__ __forceinline__ int draw_tickets(const PagedAttnArgs& a, const Pending (&pend)[2], int n, int* last) {
  unsigned* const tickets = static_cast<unsigned*>(a.workspace) + a.ticket0;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if ((int)threadIdx.x < n) {
    const PlanParts pp = {threadIdx.x ? pend[1].parts.first : pend[0].parts.first,
                          threadIdx.x ? pend[1].parts.count : pend[0].parts.count};
    const bool is = __hip_atomic_fetch_add(tickets + pp.first, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                    (unsigned)(pp.count - 1);
    if (is) __hip_atomic_store(tickets + pp.first, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last[threadIdx.x] = is;
  }
  __syncthreads();
  return (n > 0 && uniform(last[0]) ? 1 : 0) | (n > 1 && uniform(last[1]) ? 2 : 0);
}

// The partial results as one buffer; byte offset of workgroup w's part.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t parts_of(const PagedAttnArgs& a) {
  const int at = 4 * kPagedTicketWords + a.part0;
  return rsrc(static_cast<char*>(a.workspace) + at, HK_PAGED_WORKSPACE - at);
}

// The rows [r0, r0 + rows) of kv head g once more, a wave per row, 64 slots at a
// time: a lane per slot for the scores, D / 64 dimensions per lane for P @ V.
// For tasks whose tiles hold an infinity or NaN that only some of their rows
// see: in a matrix product it would reach the others as 0 * inf.  It is right
// and slow: one infinity among the newest 300 values of one kv head makes a
// piece of 701 tokens over 3003 slots take 41 ms instead of 0.07, one among the
// newest 1000 a piece of 2039 tokens over 30011 slots 542 ms instead of 1.1, one
// in each of 16 chats' last tokens a check of five 10 ms instead of 0.02.
template <int D, bool E4M3>
__device__ __forceinline__ float pool_value(const char* p, int i) {
  if constexpr (E4M3) return __builtin_amdgcn_cvt_f32_fp8(ldg(reinterpret_cast<const uint8_t*>(p) + i), 0);
  return bf16_to_f32(ldg(reinterpret_cast<const uint16_t*>(p) + i));
}
template <int D, bool E4M3>
__device__ __forceinline__ void rows_again(const PagedAttnArgs& a, const Entry& en, int g, int r0, int rows) {
  constexpr int kPer = D / 64;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), shift = a.c.page_shift;
  const int32_t* const table = a.c.table + (int64_t)max(en.seq, 0) * a.c.width;
  const float ks = score_scale<E4M3>(a, g), vs = E4M3 ? a.c.v_scale[g] : 1.0f;
  for (int r = r0 + wave; r < r0 + rows; r += kWaves) {
    const int tok = plan_div(r, a.by_group), h = g * a.group + r - tok * a.group, p = en.e.length - en.e.count + tok;
    const int64_t row = en.row0 + tok;
    const uint16_t* q = a.q + row * a.q_stride + h * D;
    float m = -INFINITY, l = 0.0f, o[kPer] = {};
    for (int j0 = a.window > 0 ? max(0, p - a.window + 1) : 0; j0 <= p; j0 += 64) {
      const int j = j0 + lane, page = j <= p ? table[j >> shift] : -1;
      const bool on = (unsigned)page < (unsigned)a.c.pages;
      const int64_t off = on ? page * a.c.page_bytes + (((int64_t)g << shift) + (j & ((1 << shift) - 1))) * D * a.c.elt : 0;
      float d = 0.0f;
      if (on)
        for (int i = 0; i < D; ++i) d = fmaf(bf16_to_f32(q[i]), pool_value<D, E4M3>(a.c.k + off, i), d);
      const float sc = on ? d * ks : -INFINITY;
      const float m_new = fmaxf(m, group_max<64>(sc)), f = __builtin_amdgcn_exp2f(m - finite_max(m_new));
      const float e = on ? __builtin_amdgcn_exp2f(sc - finite_max(m_new)) : 0.0f;
      l = l * f + group_sum<64>(e);
      m = m_new;
#pragma unroll
      for (int k = 0; k < kPer; ++k) o[k] *= f;
      for (int i = 0; i < 64; ++i) {
        if (!__shfl((int)on, i, 64)) continue;
        const float x = __shfl(e, i, 64);
        const int64_t at = (int64_t)((uint64_t)(uint32_t)__shfl((int)(off >> 32), i, 64) << 32 | (uint32_t)__shfl((int)off, i, 64));
#pragma unroll
        for (int k = 0; k < kPer; ++k) o[k] = fmaf(x, pool_value<D, E4M3>(a.c.v + at, lane + 64 * k), o[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      a.out[row * a.out_stride + h * D + lane + 64 * k] = (uint16_t)f32_to_bf16(l == 0.0f ? 0.0f : o[k] / l * vs);
    if (a.lse && lane == 0) a.lse[row * a.q_heads + h] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

// ---- up to 64 rows: the waves share the slots ----
//
// A wave takes 32 slots at a time: K straight into the MFMA's left operand
// (lane L: slot L % 16, 16 bytes at dimension 8 (L / 16) + ..), V into the
// wave's own LDS rows, which ds_read_b64_tr_b16 reads transposed.  The four
// waves of a workgroup run on their own (slots 32 w .. of each block of 128,
// no barrier) with their own maxima and sums, and meet at the end of a task.
// NQ groups of 16 rows are the MFMA's 16 columns each.
//
// Memory bounds it: a tile reads every slot once (so entries of up to 16 NQ rows
// read theirs once, others once per tile), with streaming loads (7.1 TB/s in a
// plain read of 4 GiB, 6.1 without), and a tile's K and V (16 to 64 KiB per
// workgroup) are always on the way, asked for as soon as their registers are
// free.  48 chats of up to 9001 slots, 8 kv heads of 128, bf16 (549 MB):
// 95.3 us, 78 at 7.1 TB/s, 6.8 TB/s inside the loop; the plan before it takes 3
// us, the workgroups' unequal ends 5 to 10, tickets and joins 7.  190 chats in
// e4m3 (270 MB): 62 us, 38 at that rate.  16 chats' check of five tokens (35
// rows in two tiles, 15 MB read twice): 20 us, of these 3 to plan, 4 in the loop,
// 8 to join some twenty parts of a tile.  One tile of 64 rows instead took 24.5
// us there, and 45.2 against 47.3 for 100 such chats of up to 9000 slots: it is
// not kept for that twentieth.  One chat of 71 slots: 6.5 us, a launch alone 3.8.
constexpr int kNarrowSlots = 32;

template <int D, bool E4M3, int NQ>
struct Narrow {
  static constexpr int kRows = 16 * NQ;
  static constexpr int kRowBytes = D * (E4M3 ? 1 : 2);
  static constexpr int kSteps = D / 32;                    // MFMAs of a score
  static constexpr int kKLoads = kRowBytes / 64;           // per 16 slots
  static constexpr int kVLoads = kRowBytes / 64;           // per 16 slots
  static constexpr int kDims = D / 16;
  static constexpr int kPitch = D + 4;                     // floats of a row of O in LDS
  static constexpr int kLds = kNarrowSlots * D * 2 > 16 * kPitch * 4 ? kNarrowSlots * D * 2 : 16 * kPitch * 4;  // of a wave
  static constexpr int kSmem = kWaves * kLds;
  // floats of a task's partial result: O [rows][D], max [rows], sum [rows]
  static constexpr int kPart = kRows * (D + 2);
};

// The position of 16-byte chunk c of V row r in LDS: c ^ key (an even number),
// so that the rows of a transposed read, 32 bytes of each of eight, lie in
// different banks, four by four and all eight.
template <int D>
__device__ __forceinline__ int v_key(int r) {
  return D == 128 ? 2 * (r & 7) : 2 * (((r >> 1) & 3) ^ (2 * (r & 1)));
}

// Workgroups per CU: what the registers of the loop let on it.  The e4m3 form at
// head_dim 128 keeps seven words a lane in scratch for its third (numbers of a
// task, read once per task; none in the loop over blocks).  With two, which
// need no scratch, 190 chats take 58.7 us where three take 61.8, 48 chats of up
// to 9001 slots 54.9 and 57.4.
constexpr int narrow_per_cu(int d, bool e4m3, int nq) { return nq == 2 ? 2 : d == 64 ? 4 : e4m3 ? 3 : 2; }

template <int D, bool E4M3, int NQ>
__device__ __forceinline__ void narrow_tasks(const PagedAttnArgs& a, char* smem) {
  using N = Narrow<D, E4M3, NQ>;
  char (&lds)[kWaves][N::kLds] = *reinterpret_cast<char (*)[kWaves][N::kLds]>(smem);
  __shared__ float wm[kWaves][N::kRows], wl[kWaves][N::kRows];
  __shared__ int last[2], again[kWaves];
  constexpr int kJoin = D * NQ == 256 ? 8 : 16;  // parts at a time
  static_assert(4 * kJoin * N::kRows <= kWaves * N::kLds, "the weights fit the waves' LDS rows");
  const PlanShape shape = {a.c.kv_heads, a.group, a.by_group, a.window, N::kRows, kWaves * kNarrowSlots, kBlockCost, kNarrowTaskCost};
  Run run;
  Task t;
  if (!plan_run<false>(a, shape, 1, run) || !next_task<false>(a, shape, run, t)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, quad = lane >> 4;
  const int shift = a.c.page_shift, mask = (1 << shift) - 1;
  char* const mylds = lds[wave];
  const __amdgpu_buffer_rsrc_t parts = parts_of(a);
  Pending pend[2];
  int pending = 0;
  // four dimensions of a finished row, and its lse
  auto finish = [&](const Entry& en, int g, int r, int d, const f32x4& x, float m, float l) {
    const int tok = plan_div(r, a.by_group), h = g * a.group + r - tok * a.group;
    const int64_t row = en.row0 + tok;
    const float f = l == 0.0f ? 0.0f : (E4M3 ? a.c.v_scale[g] : 1.0f) / l;
    u32x2_t y = {f32x2_to_bf16x2(x[0] * f, x[1] * f), f32x2_to_bf16x2(x[2] * f, x[3] * f)};
    if (l == 0.0f) y = u32x2_t{0u, 0u};
    stg(reinterpret_cast<u32x2_t*>(a.out + row * a.out_stride + h * D + d), y);
    if (a.lse && d == 0) stg(a.lse + row * a.q_heads + h, l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2);
  };

  u32x4 kr[2][N::kKLoads], vr[2][N::kVLoads];
  int there = 0, there_next = 0;  // bit h: slots 16 h .. of the tile have a page
  int64_t at[2];
  int bytes[2], page[2];
  // the tile's pages, asked for a tile before their rows
  auto find_pages = [&](const Task& t, int s0) {
    const int s_end = min(t.kb1 * kWaves * kNarrowSlots, t.seen);

#pragma unroll
    for (int h = 0; h < 2; ++h) page[h] = s0 + 16 * h < s_end ? table_at(t.table, (s0 + 16 * h) >> shift) : -1;
  };
  // slots [s0, s0 + 32) of the tile, read through resources that end with the
  // page's rows below t.seen: later slots, and absent pages, read zero
  auto find_tile = [&](const Task& t, int s0) {
    there_next = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int s = s0 + 16 * h;
      const bool on = (unsigned)page[h] < (unsigned)a.c.pages;
      if (on) there_next |= 1 << h;
      bytes[h] = on ? min(16, t.seen - s) * N::kRowBytes : 0;
      at[h] = on ? page[h] * a.c.page_bytes + (((int64_t)t.g << shift) + (s & mask)) * N::kRowBytes : 0;
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < N::kVLoads; ++i)
        vr[h][i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc(a.c.v + at[h], bytes[h]), 16 * lane + 1024 * i, 0, kStream);
  };
  auto load_k = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < N::kKLoads; ++i)
        kr[h][i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc(a.c.k + at[h], bytes[h]),
                                                         col * N::kRowBytes + 16 * quad + 64 * i, 0, kStream);
  };

  // the first loads of a task
  auto begin = [&](const Task& t) {
    const int s0 = (t.kb0 * kWaves + wave) * kNarrowSlots;
    if (s0 >= min(t.kb1 * kWaves * kNarrowSlots, t.seen)) return;
    find_pages(t, s0);
    find_tile(t, s0);
    load_v();
    load_k();
    find_pages(t, s0 + kWaves * kNarrowSlots);
  };

  // Of a CU's workgroups the hardware serves the oldest first, and the others end
  // last.  A wave's priority falls with its progress, through the four levels
  // three times: who is behind goes first (190 chats, e4m3: 62.0 us, without 64.2;
  // 48 chats 95.4 and 96.2).
  const int stretch = max(1, (int)min(run.r.per, (int64_t)INT32_MAX) / (12 * kBlockCost));
  int level = 3, until = stretch;
  auto step_priority = [&]() {
    if (--until > 0) return;
    until = stretch;
    level = level > 0 ? level - 1 : 3;
    if (level == 3) __builtin_amdgcn_s_setprio(3);
    else if (level == 2) __builtin_amdgcn_s_setprio(2);
    else if (level == 1) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
  };
  __builtin_amdgcn_s_setprio(3);

  begin(t);
  for (;;) {
    const int r0 = t.r0, rows = t.rows, pos0 = t.pos0, g = t.g;
    const float ks = score_scale<E4M3>(a, g);

    // this lane's rows: position, and Q as the right operand (row col of each
    // group, dimensions as the K loads give them)
    int pos[NQ], low[NQ];  // (low, pos] are the slots that the row sees
    bf16x8 qf[NQ][N::kSteps];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = r0 + 16 * n + col, tok = plan_div(r, a.by_group);
      const bool ok = 16 * n + col < rows;
      pos[n] = ok ? pos0 + tok : -1;
      low[n] = a.window > 0 ? pos[n] - a.window : -1;
      const uint16_t* q = a.q + (t.entry.row0 + (ok ? tok : 0)) * a.q_stride + (g * a.group + (ok ? r - tok * a.group : 0)) * D;
#pragma unroll
      for (int s = 0; s < N::kSteps; ++s) {
        const int d = E4M3 ? 64 * (s / 2) + 16 * quad + 8 * (s % 2) : 32 * s + 8 * quad;
        qf[n][s] = __builtin_bit_cast(bf16x8, load16(q + d));
      }
    }
    // Q is there before the loop: a wait inside it would be one for the K and V
    // loads in flight too
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int s = 0; s < N::kSteps; ++s) settle(qf[n][s]);

    float m_run[NQ], l_run[NQ];
    f32x4 o[NQ][N::kDims];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m_run[n] = -INFINITY;
      l_run[n] = 0.0f;
#pragma unroll
      for (int d = 0; d < N::kDims; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    bool poison = false;
    const int s_end = min(t.kb1 * kWaves * kNarrowSlots, t.seen);
    for (int s0 = (t.kb0 * kWaves + wave) * kNarrowSlots; s0 < s_end; s0 += kWaves * kNarrowSlots) {
      step_priority();
      there = there_next;
      const bool more = s0 + kWaves * kNarrowSlots < s_end;
      // V into LDS (the reads of the tile before are done: their values have
      // been used).  Where not every row sees every slot, an infinity or NaN
      // among the values is noted for rows_again.
      const int tok0 = plan_div(r0, a.by_group), tok1 = plan_div(r0 + rows - 1, a.by_group);
      const bool whole = s0 + kNarrowSlots - 1 <= pos0 + tok0 && there == 3 &&
                         (a.window == 0 || s0 > pos0 + tok1 - a.window);
      bool bad = false;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < N::kVLoads; ++i) {
          const int b = 16 * lane + 1024 * i, r = 16 * h + b / N::kRowBytes, c = b % N::kRowBytes / 16;
          char* row = mylds + r * D * 2;
          if constexpr (E4M3) {
            const u32x4 raw = vr[h][i];
            const u32x2_t x0 = e4m3_bf16(raw[0]), x1 = e4m3_bf16(raw[1]), x2 = e4m3_bf16(raw[2]), x3 = e4m3_bf16(raw[3]);
            const u32x4 lo = {x0.x, x0.y, x1.x, x1.y}, hi = {x2.x, x2.y, x3.x, x3.y};
            *reinterpret_cast<u32x4*>(row + 16 * ((2 * c) ^ v_key<D>(r))) = lo;
            *reinterpret_cast<u32x4*>(row + 16 * ((2 * c + 1) ^ v_key<D>(r))) = hi;
            if (!whole) bad |= not_finite(lo) || not_finite(hi);
          } else {
            *reinterpret_cast<u32x4*>(row + 16 * (c ^ v_key<D>(r))) = vr[h][i];
            if (!whole) bad |= not_finite(vr[h][i]);
          }
        }
      // the next tile's loads go out as soon as their registers are free
      if (more) {
        find_tile(t, s0 + kWaves * kNarrowSlots);
        load_v();
        find_pages(t, s0 + 2 * kWaves * kNarrowSlots);
      }
      // S^T: lane holds slots s0 + 16 h + 4 quad + r of row col
      f32x4 sv[NQ][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) sv[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < N::kSteps; ++s) {
          bf16x8 kf;
          if constexpr (E4M3) {
            const u32x4 raw = kr[h][s / 2];
            const u32x2_t lo = e4m3_bf16(raw[2 * (s % 2)]), hi = e4m3_bf16(raw[2 * (s % 2) + 1]);
            kf = __builtin_bit_cast(bf16x8, u32x4{lo.x, lo.y, hi.x, hi.y});
          } else {
            kf = __builtin_bit_cast(bf16x8, kr[h][s]);
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) sv[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][s], sv[n][h], 0, 0, 0);
        }
      }
      if (more) load_k();

      // a row sees slot s.  No && and || here: the compiler made branches of
      // them, and in a form with four groups of rows the first group's
      // mask was wrong (the test with a window of one slot shows it).
      auto sees = [&](int n, int s) {
        return (s <= pos[n]) & (s > low[n]) & (bool)((there >> ((s >> 4) & 1)) & 1);
      };
      poison |= bad;
      bf16x8 pf[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sv[n][h][r] = (whole | sees(n, s0 + 16 * h + 4 * quad + r)) ? sv[n][h][r] : -INFINITY;
            mx = fmaxf(mx, sv[n][h][r]);
          }
        const float m_new = fmaxf(m_run[n], quad_max(mx) * ks), m_use = finite_max(m_new);
        const float alpha = __builtin_amdgcn_exp2f(m_run[n] - m_use);
        float p[8], rs = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[n][e >> 2][e & 3], ks, -m_use));
          rs += p[e];
        }
        l_run[n] = l_run[n] * alpha + rs;
        m_run[n] = m_new;
        if (__any(alpha != 1.0f)) {
#pragma unroll
          for (int d = 0; d < N::kDims; ++d) o[n][d] *= alpha;
        }
        pf[n] = __builtin_bit_cast(bf16x8, u32x4{f32x2_to_bf16x2(p[0], p[1]), f32x2_to_bf16x2(p[2], p[3]),
                                                 f32x2_to_bf16x2(p[4], p[5]), f32x2_to_bf16x2(p[6], p[7])});
      }
      {
        // k index 8 quad + e of the product stands for slot 16 (e / 4) + 4 quad
        // + e % 4, the probabilities this lane holds; lane col of a group of 16
        // reads 4 slots of dimension 16 d + col
        const int ra = 4 * quad + (col >> 2), rb = ra + 16;
        const char* pa = mylds + ra * D * 2 + 16 * ((col & 3) >> 1) + 8 * (col & 1);
        const char* pb = mylds + rb * D * 2 + 16 * ((col & 3) >> 1) + 8 * (col & 1);
#pragma unroll
        for (int d = 0; d < N::kDims; ++d) {
          const v4s16 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) v4s16*)(pa + 16 * ((2 * d) ^ v_key<D>(ra))));
          const v4s16 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) v4s16*)(pb + 16 * ((2 * d) ^ v_key<D>(rb))));
          const u32x2_t w0 = __builtin_bit_cast(u32x2_t, t0), w1 = __builtin_bit_cast(u32x2_t, t1);
          const bf16x8 vf = __builtin_bit_cast(bf16x8, u32x4{w0.x, w0.y, w1.x, w1.y});
#pragma unroll
          for (int n = 0; n < NQ; ++n) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n], o[n][d], 0, 0, 0);
        }
      }
    }

    // the next task's first loads are under way while this one ends
    const Task done = t;
    const bool more_tasks = next_task<false>(a, shape, run, t);
    if (more_tasks) begin(t);

    // the waves' results meet: maxima and sums, then O through LDS 16 rows at a time
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float l = quad_sum(l_run[n]);
      if (quad == 0) {
        wm[wave][16 * n + col] = m_run[n];
        wl[wave][16 * n + col] = l;
      }
    }
    {
      const int any = __any(poison);
      if (lane == 0) again[wave] = any;
    }
    const bool cut = done.cut;
    const int slot = plan_slot(done.parts, run.r.w) * (N::kPart * 4);
    constexpr int kPer = D / 16;  // outputs of a thread: dimensions kPer (tid % 16) .. of row tid / 16
    const int orow = tid >> 4, od = kPer * (tid & 15);
    bool note = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      if (16 * n >= rows) break;
      if (n > 0) __syncthreads();
      float* ow = reinterpret_cast<float*>(mylds) + col * N::kPitch + 4 * quad;
#pragma unroll
      for (int d = 0; d < N::kDims; ++d) *reinterpret_cast<f32x4*>(ow + 16 * d) = o[n][d];
      __syncthreads();
      note = again[0] | again[1] | again[2] | again[3];
      const int r = 16 * n + orow;
      if (r >= rows) continue;
      float m = wm[0][r], l = 0.0f, x[kPer] = {};
#pragma unroll
      for (int v = 1; v < kWaves; ++v) m = fmaxf(m, wm[v][r]);
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        const float f = __builtin_amdgcn_exp2f(wm[v][r] - finite_max(m));
        l = fmaf(wl[v][r], f, l);
        const float* src = reinterpret_cast<const float*>(lds[v]) + orow * N::kPitch + od;
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(src + i);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[i + k] = fmaf(y[k], f, x[i + k]);
        }
      }
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        const f32x4 y = {x[i], x[i + 1], x[i + 2], x[i + 3]};
        if (cut)
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), parts, slot + 4 * (r * D + od + i), 0, kSc1);
        else if (!note)
          finish(done.entry, g, r0 + r, od + i, y, m, l);
      }
      if (cut && (tid & 15) == 0) {
        // (a NaN in the place of a maximum, which none is, passes the note on)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(note ? NAN : m), parts, slot + 4 * (N::kRows * D + r), 0, kSc1);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l), parts, slot + 4 * (N::kRows * (D + 1) + r), 0, kSc1);
      }
    }
    __syncthreads();  // the waves' V rows are free again
    if (!cut && note) rows_again<D, E4M3>(a, done.entry, g, r0, rows);
    if (cut) {
      const Pending p = {done.parts, done.entry, g, done.tile};
      if (pending == 0) pend[0] = p; else pend[1] = p;
      ++pending;
    }
    if (!more_tasks) break;
  }
  __builtin_amdgcn_s_setprio(0);

  const int join = pending ? draw_tickets(a, pend, pending, last) : 0;
  // joins a task's parts, J at a time: all their loads go out at once, the
  // maxima and sums give each row's weights of the parts (kRowThreads threads
  // per row), and a thread adds up kItems words of four dimensions
  constexpr int kQuads = D / 4, kItems = N::kRows * kQuads / kThreads, kRowThreads = kThreads / N::kRows;
  float (&weight)[kJoin][N::kRows] = *reinterpret_cast<float (*)[kJoin][N::kRows]>(&lds[0][0]);
  auto join_task = [&](const Pending& p, auto steps) {
    constexpr int J = decltype(steps)::value, kMine = (J + kRowThreads - 1) / kRowThreads;
    const PlanParts pp = p.parts;
    const int r0 = p.tile * N::kRows, rows = min(N::kRows, p.entry.e.count * a.group - r0);
    const int row = tid / kRowThreads, sub = tid % kRowThreads;
    f32x4 x[kItems] = {};
    float m = -INFINITY, l = 0.0f;  // of row `row`, in each of its threads
    bool note = false;
    for (int k0 = 0; k0 < pp.count; k0 += J) {
      auto part = [&](int k) { return plan_slot(pp, pp.first + min(k0 + k, pp.count - 1)) * (N::kPart * 4); };
      float pm[kMine], pl[kMine];
      u32x4 y[kItems][J];
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int at = part(sub + k * kRowThreads);
        // (of rows that the task has not, words that nobody wrote: not used)
        pm[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(parts, at + 4 * (N::kRows * D + row), 0, kSc1));
        pl[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(parts, at + 4 * (N::kRows * (D + 1) + row), 0, kSc1));
      }
#pragma unroll
      for (int k = 0; k < J; ++k)
#pragma unroll
        for (int i = 0; i < kItems; ++i)
          y[i][k] = __builtin_amdgcn_raw_buffer_load_b128(
              parts, (tid + i * kThreads) / kQuads < rows ? part(k) + 16 * (tid + i * kThreads) : kNowhere, 0, kSc1);
      float m_new = m;
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        m_new = fmaxf(m_new, pm[k]);
        note |= pm[k] != pm[k];
      }
      m_new = group_max<kRowThreads>(m_new);
      const float f = __builtin_amdgcn_exp2f(m - finite_max(m_new));
      float ls = 0.0f;
      __syncthreads();  // (the weights before have been read)
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int i = sub + k * kRowThreads;
        const bool on = i < J && k0 + i < pp.count;
        const float e = on ? __builtin_amdgcn_exp2f(pm[k] - finite_max(m_new)) : 0.0f;
        ls += on ? pl[k] * e : 0.0f;
        if (i < J) weight[i][row] = e;
      }
      l = l * f + group_sum<kRowThreads>(ls);
      m = m_new;
      if (sub == 0) wm[0][row] = m, wl[0][row] = l, wm[1][row] = f;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int r = (tid + i * kThreads) / kQuads;
        x[i] *= wm[1][r];
#pragma unroll
        for (int k = 0; k < J; ++k) {
          const float e = weight[k][r];
#pragma unroll
          for (int c = 0; c < 4; ++c) x[i][c] = k0 + k < pp.count ? fmaf(__uint_as_float(y[i][k][c]), e, x[i][c]) : x[i][c];
        }
      }
    }
    // (a note is in the first row of a part, which is always there)
    if (tid == 0) again[0] = 0;
    __syncthreads();
    if (row == 0 && note) again[0] = 1;
    __syncthreads();
    if (again[0]) {
      rows_again<D, E4M3>(a, p.entry, p.head, r0, rows);
      return;
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = (tid + i * kThreads) / kQuads, d = 4 * ((tid + i * kThreads) % kQuads);
      if (r < rows) finish(p.entry, p.head, r0 + r, d, x[i], wm[0][r], wl[0][r]);
    }
  };
  for (int j = 0; j < 2; ++j) {
    if (!((join >> j) & 1)) continue;
    const Pending p = j ? pend[1] : pend[0];
    __syncthreads();  // (wm and wl of another task have been read)
    if (p.parts.count <= 4)
      join_task(p, std::integral_constant<int, 4>());
    else
      join_task(p, std::integral_constant<int, kJoin>());
  }
}

// ---- more rows: the waves share the rows ----
//
// A workgroup takes a tile of 128 rows, a wave 32 of them (the columns of
// v_mfma_f32_32x32x16_bf16), and goes through the slots 64 at a time.  K and V
// come through registers into two LDS buffers, a block ahead, one barrier per
// block.
//
// Products bound it, and what goes on beside them: a 2039-token piece over
// 30011 slots, 32 q heads of 128 on 8 (0.97 TFLOP), takes 1075 to 1145 us from
// card to card, 850 to 900 TFLOP/s (e4m3 1052 where bf16 took 1102), and half as
// many products at head_dim 64 take 701 (e4m3 692), 691 TFLOP/s; a large matrix
// product reaches 1160.  At head_dim 128 the bf16 forms keep 11 to 13 words a lane
// in scratch: numbers of a task, read once per task, none in the loop over blocks.
// MFMA is busy 41% of the SIMDs' cycles, VALU
// (exponentials, maxima, conversions) about as long; without the exponentials it
// would take 5% less, without the staging of K and V 21%, without P @ V 26%: no
// one of them is the limit.  LDS has no bank conflicts, and L2 misses are
// 3.5% of the requests.  32 rows per wave keep O and P in registers at two
// workgroups per CU; 64 rows per wave took 2360 us where 32 took 1357.
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kWideSlots = 64;

template <int D>
struct Wide {
  static constexpr int kRows = 128;
  static constexpr int kBuf = kWideSlots * D;  // bf16 of one of K, V
  static constexpr int kSmem = 4 * kBuf * 2;
  // floats of a part: O, max and sum per lane
  static constexpr int kLaneFloats = D / 2 + 2;
  static constexpr int kPart = kThreads * kLaneFloats;
};

// Positions of the 16-byte chunks of K and V rows: a K fragment read is one
// chunk of 32 rows, a transposed V read 32 bytes of each of four rows twice.
template <int D>
__device__ __forceinline__ int wide_k_key(int r) {
  return D == 128 ? r & 15 : (r & 7) ^ ((r >> 3) & 1);
}
template <int D>
__device__ __forceinline__ int wide_v_key(int r) {
  return D == 128 ? 2 * (2 * (r & 1) + 5 * ((r >> 1) & 1)) : 2 * (r & 3);
}

__device__ __forceinline__ float half_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Workgroups per CU: registers at head_dim 64 let three on it.
constexpr int wide_per_cu(int d) { return d == 64 ? 3 : 2; }

template <int N>
using At = std::integral_constant<int, N>;

template <int D, bool E4M3>
__device__ __forceinline__ void wide_tasks(const PagedAttnArgs& a, char* smem) {
  using W = Wide<D>;
  constexpr int kRowBytes = D * (E4M3 ? 1 : 2), kLoads = kRowBytes / 64, kSteps = D / 16, kDims = D / 32;
  uint16_t (&ks_lds)[2][W::kBuf] = *reinterpret_cast<uint16_t (*)[2][W::kBuf]>(smem);
  uint16_t (&vs_lds)[2][W::kBuf] = *reinterpret_cast<uint16_t (*)[2][W::kBuf]>(smem + W::kSmem / 2);
  // of each 16 slots of a block: bit 0: they have a page, bit 1: an infinity or
  // NaN among the values, where not every row sees them all
  __shared__ __attribute__((aligned(16))) int note_lds[2][kWaves];
  __shared__ int last[2], again[kWaves];
  constexpr int kQuads = D / 8;  // 16-byte words of a part's O per lane
  const PlanShape shape = {a.c.kv_heads, a.group, a.by_group, a.window, W::kRows, kWideSlots, kBlockCost, kWideTaskCost};
  Run run;
  Task t;
  if (!plan_run<true>(a, shape, 4, run) || !next_task<true>(a, shape, run, t)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, half = lane >> 5;
  const int shift = a.c.page_shift, mask = (1 << shift) - 1;
  const __amdgpu_buffer_rsrc_t parts = parts_of(a);
  Pending pend[2];
  int pending = 0;
  // the finished rows of a tile, and their lse
  auto finish = [&](const Entry& en, int g, int r0, int rows, const f32x16 (&o)[kDims], float m, float l) {
    const int at = 32 * wave + col;
    if (at >= rows) return;
    const int tok = plan_div(r0 + at, a.by_group), h = g * a.group + (r0 + at) - tok * a.group;
    const int64_t row = en.row0 + tok;
    const float f = l == 0.0f ? 0.0f : (E4M3 ? a.c.v_scale[g] : 1.0f) / l;
    uint16_t* dst = a.out + row * a.out_stride + h * D + 4 * half;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x16& x = o[d];
        u32x2_t y = {f32x2_to_bf16x2(x[4 * i] * f, x[4 * i + 1] * f), f32x2_to_bf16x2(x[4 * i + 2] * f, x[4 * i + 3] * f)};
        if (l == 0.0f) y = u32x2_t{0u, 0u};
        stg(reinterpret_cast<u32x2_t*>(dst + 32 * d + 8 * i), y);
      }
    if (a.lse && half == 0) stg(a.lse + row * a.q_heads + h, l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2);
  };

  // wave w loads slots 16 w .. of a block (one page's): resources that end
  // with the rows below t.seen, so later slots and absent pages read zero
  u32x4 kr[kLoads], vr[kLoads];
  int page, there;
  auto find_page = [&](const Task& t, int s0) {  // asked for a block before its rows
    const int s = s0 + 16 * wave;
    page = s < t.seen ? table_at(t.table, s >> shift) : -1;
  };
  auto load_block = [&](const Task& t, int s0) {
    const int s = s0 + 16 * wave;
    const bool on = (unsigned)page < (unsigned)a.c.pages;
    there = on;
    const int bytes = on ? min(16, t.seen - s) * kRowBytes : 0;
    const int64_t at = on ? page * a.c.page_bytes + (((int64_t)t.g << shift) + (s & mask)) * kRowBytes : 0;
    const __amdgpu_buffer_rsrc_t kres = rsrc(a.c.k + at, bytes), vres = rsrc(a.c.v + at, bytes);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) kr[i] = __builtin_amdgcn_raw_buffer_load_b128(kres, 16 * lane + 1024 * i, 0, 0);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) vr[i] = __builtin_amdgcn_raw_buffer_load_b128(vres, 16 * lane + 1024 * i, 0, 0);
  };
  // the first loads of a task
  auto begin = [&](const Task& t) {
    if (t.kb0 >= t.kb1) return;
    find_page(t, t.kb0 * kWideSlots);
    load_block(t, t.kb0 * kWideSlots);
    find_page(t, (t.kb0 + 1) * kWideSlots);
  };

  begin(t);
  for (;;) {
    const int r0 = t.r0, rows = t.rows, pos0 = t.pos0, g = t.g, kb0 = t.kb0, kb1 = t.kb1;
    const float ks = score_scale<E4M3>(a, g);
    // the wave's rows [w0, w1) of the tile, and the positions they span
    const int w0 = wave * 32, w1 = min(rows, w0 + 32);
    const int wave_lo = pos0 + plan_div(r0 + w0, a.by_group), wave_hi = w1 > w0 ? pos0 + plan_div(r0 + w1 - 1, a.by_group) : -1;
    const int tile_lo = pos0 + plan_div(r0, a.by_group), tile_hi = pos0 + plan_div(r0 + rows - 1, a.by_group);

    int pos, low;  // (low, pos] are the slots that the lane's row sees
    bf16x8 qf[kSteps];
    {
      const int at = w0 + col, r = r0 + at, tok = plan_div(r, a.by_group);
      const bool ok = at < rows;
      pos = ok ? pos0 + tok : -1;
      low = a.window > 0 ? pos - a.window : -1;
      const uint16_t* q = a.q + (t.entry.row0 + (ok ? tok : 0)) * a.q_stride + (g * a.group + (ok ? r - tok * a.group : 0)) * D;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) qf[s] = __builtin_bit_cast(bf16x8, load16(q + 16 * s + 8 * half));
#pragma unroll
      for (int s = 0; s < kSteps; ++s) settle(qf[s]);  // (before the loop, as in the narrow form)
    }
    float m_run = -INFINITY, l_run = 0.0f;
    f32x16 o[kDims];
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

    // a block that every row of the tile sees whole (its pages apart)
    auto all_see = [&](int s0, int lo, int hi) {
      return s0 + kWideSlots - 1 <= lo && (a.window == 0 || s0 > hi - a.window);
    };
    auto store_block = [&](int s0, int buf) {
      bool bad = false;
      const bool whole = all_see(s0, tile_lo, tile_hi);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int b = 16 * lane + 1024 * i, r = 16 * wave + b / kRowBytes, c = b % kRowBytes / 16;
        uint16_t *krow = &ks_lds[buf][r * D], *vrow = &vs_lds[buf][r * D];
        if constexpr (E4M3) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x2_t k0 = e4m3_bf16(kr[i][2 * e]), k1 = e4m3_bf16(kr[i][2 * e + 1]);
            *reinterpret_cast<u32x4*>(krow + 8 * ((2 * c + e) ^ wide_k_key<D>(r))) = u32x4{k0.x, k0.y, k1.x, k1.y};
            const u32x2_t v0 = e4m3_bf16(vr[i][2 * e]), v1 = e4m3_bf16(vr[i][2 * e + 1]);
            const u32x4 v = {v0.x, v0.y, v1.x, v1.y};
            *reinterpret_cast<u32x4*>(vrow + 8 * ((2 * c + e) ^ wide_v_key<D>(r))) = v;
            if (!whole) bad |= not_finite(v);
          }
        } else {
          *reinterpret_cast<u32x4*>(krow + 8 * (c ^ wide_k_key<D>(r))) = kr[i];
          *reinterpret_cast<u32x4*>(vrow + 8 * (c ^ wide_v_key<D>(r))) = vr[i];
          if (!whole) bad |= not_finite(vr[i]);
        }
      }
      const int any = __any(bad);
      if (lane == 0) note_lds[buf][wave] = there | any << 1;
    };

    int poison = 0;  // an infinity or NaN among values that not every row sees, for rows_again
    if (kb0 < kb1) store_block(kb0 * kWideSlots, 0);
    if (kb0 + 1 < kb1) {
      load_block(t, (kb0 + 1) * kWideSlots);
      find_page(t, (kb0 + 2) * kWideSlots);
    }
    for (int kb = kb0, buf = 0; kb < kb1; ++kb, buf ^= 1) {
      const int s0 = kb * kWideSlots;
      __syncthreads();  // the block is there, and the other buffer has been read
      // the next block, whose loads went out a block ago, goes to LDS beside this
      // one's products (behind them it cost a fifth of the time), and the loads of
      // the one after it go out
      if (kb + 1 < kb1) store_block(s0 + kWideSlots, buf ^ 1);
      if (kb + 2 < kb1) {
        load_block(t, s0 + 2 * kWideSlots);
        find_page(t, s0 + 3 * kWideSlots);
      }
      if (s0 <= wave_hi) {
        const u32x4 notes = *reinterpret_cast<const u32x4*>(note_lds[buf]);
        // The block's products in order: S^T of slots 0 .. 31 and 32 .. 63 (kSteps
        // each), then O^T with 16 slots' probabilities at a time (kDims each).
        // Their left operands come from LDS two products ahead (left to itself
        // the compiler reads one and waits for it).  At head_dim 128 the softmax
        // of a half runs between the products that do not need it, product by
        // product, with a maximum of its own; at 64, where half as many products
        // stand beside as many exponentials and a third workgroup on the CU fills
        // the gaps, it runs at once (prompt at 128: 1072 us against 1111; pieces
        // beside chats at 64: 64 against 61).
        constexpr int kQk = 2 * kSteps, kAll = kQk + 4 * kDims;
        // S^T: lane holds slots 32 t + 8 (i / 4) + 4 half + i % 4 of row col; V: k
        // index 8 half + e of product x stands for slot 16 x + 8 (e / 4) + 4 half
        // + e % 4, the probabilities that this lane holds, and a group of 16 lanes
        // reads 4 slots of 16 dimensions, transposed
        f32x16 sv[2];
        bf16x8 pf[4], left[2][2];
        const int ra = 4 * half + ((lane & 15) >> 2), dd = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        auto read_left = [&](int pair) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int x = 2 * pair + y;
            if (x < kQk) {
              const int r = 32 * (x / kSteps) + col, s = x % kSteps;
              left[pair & 1][y] = *reinterpret_cast<const bf16x8*>(&ks_lds[buf][r * D + 8 * ((2 * s + half) ^ wide_k_key<D>(r))]);
            } else {
              const int d = (x - kQk) % kDims, r1 = 16 * ((x - kQk) / kDims) + ra, r2 = r1 + 8, dim = 32 * d + dd;
              const v4s16 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) v4s16*)&vs_lds[buf][r1 * D + 8 * ((dim >> 3) ^ wide_v_key<D>(r1)) + (dim & 7)]);
              const v4s16 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) v4s16*)&vs_lds[buf][r2 * D + 8 * ((dim >> 3) ^ wide_v_key<D>(r2)) + (dim & 7)]);
              const u32x2_t w0 = __builtin_bit_cast(u32x2_t, t0), w1 = __builtin_bit_cast(u32x2_t, t1);
              left[pair & 1][y] = __builtin_bit_cast(bf16x8, u32x4{w0.x, w0.y, w1.x, w1.y});
            }
          }
        };
        auto products = [&](auto from, auto count, auto between) {
#pragma unroll
          for (int x = from; x < from + count; ++x) {
            if (x % 2 == 0) {
              __builtin_amdgcn_sched_barrier(0);
              if (x + 2 < kAll) read_left(x / 2 + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
            const bf16x8 l = left[(x / 2) & 1][x % 2];
            if (x < kQk)
              sv[x / kSteps] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(l, qf[x % kSteps], sv[x / kSteps], 0, 0, 0);
            else
              o[(x - kQk) % kDims] =
                  __builtin_amdgcn_mfma_f32_32x32x16_bf16(l, pf[(x - kQk) / kDims], o[(x - kQk) % kDims], 0, 0, 0);
            between(x - from);
          }
        };
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) sv[h][i] = 0.0f;

        // bit h: slots 16 h .. of the block have a page
        const int paged = uniform((int)((notes.x & 1) | (notes.y & 1) << 1 | (notes.z & 1) << 2 | (notes.w & 1) << 3));
        const bool whole = all_see(s0, wave_lo, wave_hi) && paged == 15;
        if (!whole) poison |= (notes.x | notes.y | notes.z | notes.w) & 2;
        auto hide = [&](int h) {
          if (whole) return;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int s = s0 + 32 * h + 8 * (i >> 2) + 4 * half + (i & 3);
            // (no && and ||, as in the narrow form: branches gave a wrong mask there)
            const bool sees = (s <= pos) & (s > low) & (bool)((paged >> ((s >> 4) & 3)) & 1);
            sv[h][i] = sees ? sv[h][i] : -INFINITY;
          }
        };
        // share `step` of `steps` of the softmax of half h: first the maximum, then
        // the exponentials in pairs.
        float alpha = 1.0f, m_use = 0.0f, sum = 0.0f, sum2 = 0.0f;
        auto soften = [&](int h, int step, int steps) {
          if (step == 0) {
            float mx = fmaxf(sv[h][0], sv[h][1]);
#pragma unroll
            for (int i = 2; i < 16; ++i) mx = fmaxf(mx, sv[h][i]);
            const float m_new = fmaxf(m_run, half_max(mx) * ks);
            m_use = finite_max(m_new);
            alpha = __builtin_amdgcn_exp2f(m_run - m_use);
            m_run = m_new;
            sum = sum2 = 0.0f;
            return;
          }
          const int i0 = 8 * (step - 1) / (steps - 1), i1 = 8 * step / (steps - 1);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i < i0 || i >= i1) continue;
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[h][2 * i], ks, -m_use));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[h][2 * i + 1], ks, -m_use));
            sum += e0;
            sum2 += e1;
            u32x4 pw = __builtin_bit_cast(u32x4, pf[2 * h + i / 4]);
            pw[i % 4] = f32x2_to_bf16x2(e0, e1);
            pf[2 * h + i / 4] = __builtin_bit_cast(bf16x8, pw);
          }
        };
        auto rescale = [&]() {
          l_run = l_run * alpha + (sum + sum2);
          if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int d = 0; d < kDims; ++d) o[d] *= alpha;
          }
        };
        __builtin_amdgcn_s_setprio(1);  // a wave in its products goes before one in its softmax (prompt: 5%)
        read_left(0);
        if constexpr (D == 128) {
          products(At<0>(), At<kSteps>(), [](int) {});
          hide(0);
          products(At<kSteps>(), At<kSteps>(), [&](int x) { soften(0, x, kSteps); });
          rescale();
          hide(1);
          products(At<kQk>(), At<2 * kDims>(), [&](int x) { soften(1, x, 2 * kDims); });
          rescale();
          products(At<kQk + 2 * kDims>(), At<2 * kDims>(), [](int) {});
        } else {
          products(At<0>(), At<kQk>(), [](int) {});
          hide(0);
          hide(1);
          __builtin_amdgcn_s_setprio(0);
          float mx = fmaxf(sv[0][0], sv[1][0]);
#pragma unroll
          for (int i = 1; i < 16; ++i) mx = fmaxf(fmaxf(mx, sv[0][i]), sv[1][i]);
          const float m_new = fmaxf(m_run, half_max(mx) * ks), m_use = finite_max(m_new);
          const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
          m_run = m_new;
          float sum = 0.0f;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            u32x4 pw;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[x / 2][8 * (x % 2) + 2 * i], ks, -m_use));
              const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[x / 2][8 * (x % 2) + 2 * i + 1], ks, -m_use));
              sum += e0;
              sum += e1;
              pw[i] = f32x2_to_bf16x2(e0, e1);
            }
            pf[x] = __builtin_bit_cast(bf16x8, pw);
          }
          l_run = l_run * alpha + sum;
          // once the running maxima settle, alpha is 1 in every lane
          if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int d = 0; d < kDims; ++d) o[d] *= alpha;
          }
          __builtin_amdgcn_s_setprio(1);
          products(At<kQk>(), At<4 * kDims>(), [](int) {});
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }

    // the next task's first loads are under way while this one ends
    const Task done = t;
    const bool more_tasks = next_task<true>(a, shape, run, t);
    if (more_tasks) begin(t);
    const bool cut = done.cut;
    l_run = half_sum(l_run);
    if (lane == 0) again[wave] = poison;
    __syncthreads();  // the buffers have been read
    const bool note = again[0] | again[1] | again[2] | again[3];
    if (cut) {
      // parts lie lane by lane: word i of thread t at 16 (i threads + t) bytes
      const int slot = plan_slot(done.parts, run.r.w) * (W::kPart * 4);
      if (wave_hi >= 0) {
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const f32x16& x = o[i / 4];
          const f32x4 y = {x[4 * (i % 4)], x[4 * (i % 4) + 1], x[4 * (i % 4) + 2], x[4 * (i % 4) + 3]};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), parts, slot + 16 * (kThreads * i + tid), 0, kSc1);
        }
        // (a NaN in the place of a maximum, which none is, passes the note on)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(note ? NAN : m_run), __float_as_uint(l_run)}, parts,
                                              slot + 16 * kThreads * kQuads + 8 * tid, 0, kSc1);
      }
      const Pending p = {done.parts, done.entry, g, done.tile};
      if (pending == 0) pend[0] = p; else pend[1] = p;
      ++pending;
    } else if (note) {
      rows_again<D, E4M3>(a, done.entry, g, r0, rows);
    } else {
      finish(done.entry, g, r0, rows, o, m_run, l_run);
    }
    __syncthreads();  // (the notes have been read)
    if (!more_tasks) break;
  }

  const int join = pending ? draw_tickets(a, pend, pending, last) : 0;
  for (int j = 0; j < 2; ++j) {
    if (!((join >> j) & 1)) continue;
    const Pending p = j ? pend[1] : pend[0];
    const PlanParts pp = p.parts;
    const int r0 = p.tile * W::kRows, rows = min(W::kRows, p.entry.e.count * a.group - r0);
    // (a wave whose rows stand at negative positions has no part)
    const bool has = p.entry.e.length - p.entry.e.count + plan_div(r0 + min(rows, 32 * (wave + 1)) - 1, a.by_group) >= 0 &&
                     rows > 32 * wave;
    float m = -INFINITY, l = 0.0f;
    f32x16 o[kDims];
    bool note = false;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    // two parts go out at once (a 2039-token piece: 1088 us, one at a time 1103)
    for (int k0 = 0; has && k0 < pp.count; k0 += 2) {
      u32x2_t ml[2];
      u32x4 y[2][kQuads];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int slot = plan_slot(pp, pp.first + min(k0 + j, pp.count - 1)) * (W::kPart * 4);
        ml[j] = __builtin_amdgcn_raw_buffer_load_b64(parts, slot + 16 * kThreads * kQuads + 8 * tid, 0, kSc1);
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
          y[j][i] = __builtin_amdgcn_raw_buffer_load_b128(parts, slot + 16 * (kThreads * i + tid), 0, kSc1);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (k0 + j >= pp.count) break;
        const float mk = __uint_as_float(ml[j].x), m_new = fmaxf(m, mk);
        const float f0 = __builtin_amdgcn_exp2f(m - finite_max(m_new)), f1 = __builtin_amdgcn_exp2f(mk - finite_max(m_new));
        note |= mk != mk;
        l = l * f0 + __uint_as_float(ml[j].y) * f1;
        m = m_new;
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            o[i / 4][4 * (i % 4) + c] = fmaf(__uint_as_float(y[j][i][c]), f1, o[i / 4][4 * (i % 4) + c] * f0);
      }
    }
    const int any = __any(note);
    if (lane == 0) again[wave] = any;
    __syncthreads();
    if (again[0] | again[1] | again[2] | again[3])
      rows_again<D, E4M3>(a, p.entry, p.head, r0, rows);
    else
      finish(p.entry, p.head, r0, rows, o, m, l);
    __syncthreads();
  }
}

// ---- kernels ----

template <int D, bool E4M3, int NQ>
__global__ __launch_bounds__(kThreads, narrow_per_cu(D, E4M3, NQ)) void paged_narrow_kernel(PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[Narrow<D, E4M3, NQ>::kSmem];
  narrow_tasks<D, E4M3, NQ>(a, smem);
}

template <int D, bool E4M3>
__global__ __launch_bounds__(kThreads, wide_per_cu(D)) void paged_wide_kernel(PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[Wide<D>::kSmem];
  wide_tasks<D, E4M3>(a, smem);
}

// Entries of a few rows (few) beside longer ones (many), each in its form: a
// workgroup takes its run of the ones, then its run of the others, without
// waiting for the workgroups that are behind.  Pieces of prompts beside chats
// with a window took 58.6 us where two launches took 65.0 (56 to 57 now); 20
// sequences of up to 9000 slots, 7 of them with 511 new tokens, head_dim 128: 287
// and 301.  (Workgroups
// that begin with the others, so that reading and products go on at the same
// time, gain no more: 60.0 and 289.)
constexpr int kCus = 256;
template <int D, bool E4M3>
__global__ __launch_bounds__(kThreads, wide_per_cu(D)) void paged_mixed_kernel(PagedAttnArgs few, PagedAttnArgs many) {
  constexpr int kSmem = Narrow<D, E4M3, 1>::kSmem > Wide<D>::kSmem ? Narrow<D, E4M3, 1>::kSmem : Wide<D>::kSmem;
  __shared__ __attribute__((aligned(16))) char smem[kSmem];
  narrow_tasks<D, E4M3, 1>(few, smem);
  __syncthreads();
  wide_tasks<D, E4M3>(many, smem);
}

// Launches: as many workgroups as the GPU holds at once.
constexpr int64_t part_bytes(long long groups, long long part) { return 2 * groups * part * 4; }
constexpr bool fits(long long groups, long long bytes) {
  return groups <= kPagedTicketWords && groups % 8 == 0 && 4ll * kPagedTicketWords + bytes <= HK_PAGED_WORKSPACE;
}
template <int D, bool E4M3, int NQ>
constexpr bool narrow_fits() {
  constexpr int groups = kCus * narrow_per_cu(D, E4M3, NQ);
  return fits(groups, part_bytes(groups, Narrow<D, E4M3, NQ>::kPart));
}
template <int D>
constexpr bool wide_fits() {  // with the narrow form's beside it
  constexpr int groups = kCus * wide_per_cu(D);
  return fits(2 * groups, part_bytes(groups, Wide<D>::kPart) + part_bytes(groups, Narrow<D, false, 1>::kPart));
}
static_assert(narrow_fits<64, false, 1>() && narrow_fits<64, true, 1>() && narrow_fits<128, false, 1>() &&
                  narrow_fits<128, true, 1>() && narrow_fits<64, false, 2>() && narrow_fits<64, true, 2>() &&
                  narrow_fits<128, false, 2>() && narrow_fits<128, true, 2>() && wide_fits<64>() && wide_fits<128>(),
              "partial results and tickets fit the workspace");

constexpr char kLaunch[] = "paged attention launch";

// Which form takes an entry goes by its rows (new tokens x heads per kv head),
// as far as max_new says.
//
// Up to 64 rows in all entries: the narrow form.  Above 32 that is two tiles, and
// it is the better one for few entries (16 chats x 35 rows, 14 heads on 2 of 64:
// 19.6 us, wide 35.1; one of 64 rows over 30011 slots, 32 heads on 8 of 128: 62
// and 123; four of 48 rows over 6011: 49 and 65), the worse one for many (100
// chats of up to 9000 slots, 35 rows of 64: 65 and 59; 48 rows of 128: 434 and
// 316; 64 rows: 448 and 318): those at head_dim 128 read more than L2 holds, and
// each tile reads it again.  Above 64 rows wide is ahead for many as well (100
// chats, 80 rows: 331, narrow 648; 112 rows of 64: 69 and 117).
//
// Long entries beside short ones: entries of up to 16 rows, a decode step's, in
// the narrow form and all others in the wide one, one launch for both.  Entries of
// 17 to 64 rows then get a 128-row tile; with a narrow launch of 32-row tiles of
// their own in front, two pieces of 511 tokens beside 24 chats x 28 rows of 64
// take 67.5 us instead of 53.5, beside 24 x 32 rows of 128 157 instead of 149,
// beside 100 of those 270 instead of 305; one for up to 64 rows costs 16 to 28 us
// more beside 24 chats of 35 rows.
//
// 17 to 32 heads per kv head: a decode step's entry has more than 16 rows, and
// gets that launch of its own.  Two pieces of 64 tokens beside 100 chats of up to
// 9000 slots, 24 heads per kv head of 128: 340 us, all wide 372; beside 24: 181
// and 179; at head_dim 64 it is behind (100 chats: 121 and 104; 24: 81 and 64).
//
// One launch for the entries of rows_min .. rows_max rows, `rows` of them at
// most as far as the caller knows.
template <int D, bool E4M3>
int narrow(const PagedAttnArgs& a, int64_t rows, hipStream_t stream) {
  if (rows <= 16) return paged_launch(kLaunch, paged_narrow_kernel<D, E4M3, 1>, kCus * narrow_per_cu(D, E4M3, 1), kThreads, stream, a);
  return paged_launch(kLaunch, paged_narrow_kernel<D, E4M3, 2>, kCus * narrow_per_cu(D, E4M3, 2), kThreads, stream, a);
}

template <int D, bool E4M3>
int launch(PagedAttnArgs a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.max_new * a.group;
  constexpr int kWideGroups = kCus * wide_per_cu(D);
  a.by_group = plan_divisor(a.group);
  a.rows_min = 1;
  a.rows_max = INT32_MAX;
  a.ticket0 = a.part0 = 0;
  if (rows <= 64) return narrow<D, E4M3>(a, rows, stream);
  // entries of a few rows beside longer ones
  const int few = a.group <= 16 ? 16 : 32;
  if (a.b.n > 1 && a.group <= few) {
    PagedAttnArgs b = a;
    b.rows_max = few;
    a.rows_min = few + 1;
    if (few == 16) {
      a.ticket0 = kWideGroups;
      a.part0 = (int)part_bytes(kWideGroups, Narrow<D, E4M3, 1>::kPart);
      return paged_launch(kLaunch, paged_mixed_kernel<D, E4M3>, kWideGroups, kThreads, stream, b, a);
    }
    if (const int rc = narrow<D, E4M3>(b, few, stream)) return rc;
  }
  return paged_launch(kLaunch, paged_wide_kernel<D, E4M3>, kWideGroups, kThreads, stream, a);
}

}  // namespace

int launch_paged_attention(const PagedAttnArgs& a, int head_dim, hipStream_t stream) {
  const bool e4m3 = a.c.elt == 1;
  if (head_dim == 64) return e4m3 ? launch<64, true>(a, stream) : launch<64, false>(a, stream);
  return e4m3 ? launch<128, true>(a, stream) : launch<128, false>(a, stream);
}

}  // namespace hk
