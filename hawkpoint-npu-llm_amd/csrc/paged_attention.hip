// Attention of a batch's new tokens over a paged KV cache (hk_paged_attention).
//
// Row (token t of an entry, head h) stands at position p = length - count + t
// and sees the slots j <= p (with a window, j > p - window) whose page exists:
//   s_j = scale (q . k_j),  m = max s_j,  l = sum exp(s_j - m)
//   out = sum exp(s_j - m) v_j / l,  lse = m + ln l
// in one pass over the slots with a running maximum and sum.  The rows of all
// query heads of a kv head are one tile's rows, so K and V are read once for
// them.  S^T = K Q^T puts a row's scores into the lanes that hold the row's
// column of P^T, the right operand of O^T = V^T P^T: the probabilities never
// leave their registers.  They are rounded to bf16 there (2^-8 of each at
// most, about what the rounding of the result costs; the three-term split of
// the prefill kernel would triple the products), scores, maxima and sums are
// float32.
//
// The work of a batch is cut into equal runs of blocks (paged_plan.h), which
// every workgroup works out by itself from the lengths on the device: a batch
// of mixed lengths fills the GPU, a captured launch fits every later length,
// and there is nothing to plan between the calls.  A task that is cut leaves
// (max, sum, O) of its parts in the workspace, and the workgroup that arrives
// last (a ticket per task, zero between launches) joins them in their order.
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
constexpr int kSc1 = 16;  // buffer access cache policy: device scope

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// ---- a workgroup's run of the work ----

struct Entry {
  int seq, row0;  // sequence (-1: none), first row
  PlanEntry e;
};
__device__ __forceinline__ Entry load_entry(const PagedAttnArgs& a, int b) {
  const int2 r = entry_rows(a.b, b), s = entry_seq(a.c, a.b, b);
  return {uniform(s.x), uniform(r.x), {uniform(s.y), uniform(r.y - r.x)}};
}

// Sum of v over the workgroup in every thread, and the sum of the threads
// before this one.
__device__ __forceinline__ int64_t scan(int64_t v, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t s = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int64_t u = __shfl_up(s, m, 64);
    if (lane >= m) s += u;
  }
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

struct Run {
  int64_t unit, end, per;
  PlanPlace place;
  Entry entry;
};

// The run of workgroup w of `groups`; false: it has none.
__device__ __forceinline__ bool plan_run(const PagedAttnArgs& a, const PlanShape& s, int w, int groups, int least,
                                         Run& run) {
  __shared__ int64_t sums[kWaves];
  __shared__ int64_t found_start;
  __shared__ int found;
  const int n = a.b.n;
  auto units = [&](int b) -> int64_t {
    if (b >= n) return 0;
    const int2 r = entry_rows(a.b, b);
    if (r.y == r.x) return 0;
    return s.heads * plan_head_units(s, {entry_seq(a.c, a.b, b).y, r.y - r.x});
  };
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
  run.per = plan_per(total, groups, least);
  run.unit = w * run.per;
  run.end = min(total, run.unit + run.per);
  if (run.unit >= run.end) return false;
  int64_t base = 0;
  for (int b0 = 0; b0 < n; b0 += kThreads) {
    int64_t chunk = 0;
    if (b0 > 0) {
      mine = units(b0 + threadIdx.x);
      before = base + scan(mine, sums, chunk);
    } else if (n > kThreads) {
      scan(mine, sums, chunk);
    }
    if (before <= run.unit && run.unit < before + mine) {
      found = b0 + threadIdx.x;
      found_start = before;
    }
    base += chunk;
  }
  __syncthreads();
  const int b = uniform(found);
  const int64_t start = uniform(found_start);
  run.entry = load_entry(a, b);
  run.place = plan_find(s, run.entry.e, b, start, run.unit - start);
  return true;
}

// On to the next task.
__device__ __forceinline__ void plan_next(const PagedAttnArgs& a, const PlanShape& s, Run& run, int units) {
  PlanPlace& p = run.place;
  p.at = 0;
  p.start += units;
  if (++p.tile < plan_tiles(s, run.entry.e)) return;
  p.tile = 0;
  if (++p.head < s.heads) return;
  p.head = 0;
  while (++p.entry < a.b.n) {
    run.entry = load_entry(a, p.entry);
    if (run.entry.e.count > 0) return;
  }
}

// Consecutive runs on one XCD (workgroups go round the eight XCDs), where they
// share K and V rows in its L2.
__device__ __forceinline__ int run_of_group() {
  const int groups = gridDim.x;  // a multiple of 8
  return (int)blockIdx.x % 8 * (groups / 8) + (int)blockIdx.x / 8;
}

// 2^(score - max): where all scores are -inf the maximum is no number to subtract.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

// Whether one of the eight bf16 values is an infinity or NaN.
__device__ __forceinline__ bool not_finite(const u32x4& v) {
  bool bad = false;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    bad |= (v[w] & 0x7f80u) == 0x7f80u || (v[w] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// Four e4m3 values as two bf16 pairs (exact: every e4m3 value is a bf16 value).
__device__ __forceinline__ u32x2_t e4m3_bf16(uint32_t w) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  constexpr uint32_t kTops = 0x07060302u;  // a float's high half is the exact bf16
  return u32x2_t{__builtin_amdgcn_perm(__float_as_uint(lo.y), __float_as_uint(lo.x), kTops),
                 __builtin_amdgcn_perm(__float_as_uint(hi.y), __float_as_uint(hi.x), kTops)};
}

// ---- up to 64 rows: the waves share the slots ----
//
// A wave takes 32 slots at a time: K straight into the MFMA's left operand
// (lane L: slot L % 16, 16 bytes at dimension 8 (L / 16) + ..), V into the
// wave's own LDS rows, which ds_read_b64_tr_b16 reads transposed.  The four
// waves of a workgroup run on their own (slots 32 w .. of each block of 128,
// no barrier) with their own maxima and sums, and meet at the end of a task.
// NQ groups of 16 rows are the MFMA's 16 columns each.
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
  static constexpr int kLds = kNarrowSlots * D * 2 > 16 * kPitch * 4 ? kNarrowSlots * D * 2 : 16 * kPitch * 4;
  // floats of a task's partial result: O [rows][D], max [rows], sum [rows]
  static constexpr int kPart = kRows * (D + 2);
};

// The position of 16-byte chunk c of V row r in LDS: c ^ key, so that the four
// rows of a transposed read lie in different banks.
template <int D>
__device__ __forceinline__ int v_key(int r) {
  return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
}

template <int D, bool E4M3, int NQ>
__global__ __launch_bounds__(kThreads, NQ == 4 ? 1 : 2) void paged_narrow_kernel(PagedAttnArgs a) {
  using N = Narrow<D, E4M3, NQ>;
  __shared__ __attribute__((aligned(16))) char lds[kWaves][N::kLds];
  __shared__ float wm[kWaves][N::kRows], wl[kWaves][N::kRows];
  __shared__ int last;
  const PlanShape shape = {a.c.kv_heads, a.group, a.window, N::kRows, kWaves * kNarrowSlots};
  const int w = run_of_group();
  Run run;
  if (!plan_run(a, shape, w, gridDim.x, 1, run)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, quad = lane >> 4;
  const int shift = a.c.page_shift, mask = (1 << shift) - 1;
  char* const mylds = lds[wave];
  float* const parts = static_cast<float*>(a.workspace) + kPagedTicketWords;
  unsigned* const tickets = static_cast<unsigned*>(a.workspace);

  while (run.unit < run.end) {
    const PlanSpan span = plan_span(shape, run.entry.e, run.place.tile);
    const int units = plan_units(span);
    const int take = (int)min((int64_t)(units - run.place.at), run.end - run.unit);
    const int g = run.place.head, r0 = run.place.tile * N::kRows;
    const int rows = min(N::kRows, run.entry.e.count * a.group - r0);
    const int pos0 = run.entry.e.length - run.entry.e.count;
    const int kb0 = span.lo + run.place.at, kb1 = span.hi > span.lo ? kb0 + take : kb0;
    const int32_t* const table = a.c.table + (int64_t)max(run.entry.seq, 0) * a.c.width;
    const float ks = (E4M3 ? a.c.k_scale[g] : 1.0f) * a.scale * kLog2e;

    // this lane's rows: position, and Q as the right operand (row col of each
    // group, dimensions as the K loads give them)
    int pos[NQ], low[NQ];  // (low, pos] are the slots that the row sees
    bf16x8 qf[NQ][N::kSteps];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = r0 + 16 * n + col, tok = r / a.group;
      const bool ok = 16 * n + col < rows;
      pos[n] = ok ? pos0 + tok : -1;
      low[n] = a.window > 0 ? pos[n] - a.window : -1;
      const uint16_t* q = a.q + (run.entry.row0 + (ok ? tok : 0)) * a.q_stride + (g * a.group + (ok ? r - tok * a.group : 0)) * D;
#pragma unroll
      for (int s = 0; s < N::kSteps; ++s) {
        const int d = E4M3 ? 64 * (s / 2) + 16 * quad + 8 * (s % 2) : 32 * s + 8 * quad;
        qf[n][s] = __builtin_bit_cast(bf16x8, load16(q + d));
      }
    }

    float m_run[NQ], l_run[NQ];
    f32x4 o[NQ][N::kDims];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m_run[n] = -INFINITY;
      l_run[n] = 0.0f;
#pragma unroll
      for (int d = 0; d < N::kDims; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    u32x4 kr[2][N::kKLoads], vr[2][N::kVLoads];
    int there = 0, there_next = 0;  // bit h: slots 16 h .. of the tile have a page
    // slots [s0, s0 + 32) of the tile, read through resources that end with the
    // page's rows below span.seen: later slots, and absent pages, read zero
    auto load_tile = [&](int s0) {
      there_next = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int s = s0 + 16 * h;
        const int page = s < span.seen ? uniform(table[s >> shift]) : -1;
        const bool on = (unsigned)page < (unsigned)a.c.pages;
        if (on) there_next |= 1 << h;
        const int bytes = on ? min(16, span.seen - s) * N::kRowBytes : 0;
        const int64_t at = on ? page * a.c.page_bytes + (((int64_t)g << shift) + (s & mask)) * N::kRowBytes : 0;
        const __amdgpu_buffer_rsrc_t kres = rsrc(a.c.k + at, bytes), vres = rsrc(a.c.v + at, bytes);
#pragma unroll
        for (int i = 0; i < N::kKLoads; ++i)
          kr[h][i] = __builtin_amdgcn_raw_buffer_load_b128(kres, col * N::kRowBytes + 16 * quad + 64 * i, 0, 0);
#pragma unroll
        for (int i = 0; i < N::kVLoads; ++i)
          vr[h][i] = __builtin_amdgcn_raw_buffer_load_b128(vres, 16 * lane + 1024 * i, 0, 0);
      }
    };

    const int s_end = min(kb1 * kWaves * kNarrowSlots, span.seen);
    int s0 = (kb0 * kWaves + wave) * kNarrowSlots;
    if (s0 < s_end) load_tile(s0);
    for (; s0 < s_end; s0 += kWaves * kNarrowSlots) {
      there = there_next;
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
      // V into LDS (the reads of the tile before are done: their values have
      // been used).  Slots that not every row sees are the only ones whose
      // values may not reach a product with 0.
      const int tok0 = r0 / a.group, tok1 = (r0 + rows - 1) / a.group;
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
      if (s0 + kWaves * kNarrowSlots < s_end) load_tile(s0 + kWaves * kNarrowSlots);

      // a row sees slot s (no branches: the lanes differ)
      auto sees = [&](int n, int s) {
        return (s <= pos[n]) & (s > low[n]) & (bool)((there >> ((s >> 4) & 1)) & 1);
      };
      const bool slow = !whole && __any(bad);
      bf16x8 pf[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sv[n][h][r] = whole | sees(n, s0 + 16 * h + 4 * quad + r) ? sv[n][h][r] : -INFINITY;
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
      if (!slow) {
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
      } else {
        // an infinity or NaN in a tile that not every row sees whole: slot by
        // slot, so that it reaches the rows that see it and no other
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          for (int j = 0; j < kNarrowSlots; ++j) {
            const u32x4 pw = __builtin_bit_cast(u32x4, pf[n]);
            const int e = 4 * (j >> 4) + (j & 3);
            const uint32_t word = e < 2 ? pw[0] : e < 4 ? pw[1] : e < 6 ? pw[2] : pw[3];
            const float mine = (e & 1) ? bf_hi(word) : bf_lo(word);
            const float pj = __shfl(mine, col + 16 * ((j >> 2) & 3), 64);
            if (sees(n, s0 + j)) {
#pragma unroll
              for (int d = 0; d < N::kDims; ++d) {
                const int dim = 16 * d + 4 * quad;
                const uint16_t* v = reinterpret_cast<const uint16_t*>(mylds + j * D * 2 + 16 * ((dim >> 3) ^ v_key<D>(j))) + (dim & 7);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[n][d][r] = fmaf(pj, bf16_to_f32(v[r]), o[n][d][r]);
              }
            }
          }
      }
    }

    // the waves' results meet: maxima and sums, then O through LDS 16 rows at a time
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float l = quad_sum(l_run[n]);
      if (quad == 0) {
        wm[wave][16 * n + col] = m_run[n];
        wl[wave][16 * n + col] = l;
      }
    }
    const bool cut = take < units;
    const PlanParts pp = plan_parts(run.place.start, units, run.per);
    const float vs = E4M3 ? a.c.v_scale[g] : 1.0f;
    constexpr int kPer = D / 16;  // outputs of a thread: dimensions kPer (tid % 16) .. of row tid / 16
    const int orow = tid >> 4, od = kPer * (tid & 15);
    // a finished row: out and lse
    auto finish = [&](int r, const float (&x)[kPer], float m, float l) {
      const int tok = (r0 + r) / a.group, h = g * a.group + (r0 + r) % a.group;
      const int64_t row = run.entry.row0 + tok;
      const float f = l == 0.0f ? 0.0f : vs / l;
      uint32_t ow[kPer / 2];
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i)
        ow[i] = l == 0.0f ? 0u : f32x2_to_bf16x2(x[2 * i] * f, x[2 * i + 1] * f);
      uint16_t* dst = a.out + row * a.out_stride + h * D + od;
      if constexpr (kPer == 8)
        stg(reinterpret_cast<u32x4*>(dst), u32x4{ow[0], ow[1], ow[2], ow[3]});
      else
        stg(reinterpret_cast<u32x2_t*>(dst), u32x2_t{ow[0], ow[1]});
      if (a.lse && (tid & 15) == 0)
        stg(a.lse + row * a.q_heads + h, l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2);
    };
    float* const mine = parts + (int64_t)plan_slot(run.place.start, w, run.per) * N::kPart;
    const __amdgpu_buffer_rsrc_t mres = rsrc(mine, N::kPart * 4);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      if (16 * n >= rows) break;
      if (n > 0) __syncthreads();
      float* ow = reinterpret_cast<float*>(mylds) + col * N::kPitch + 4 * quad;
#pragma unroll
      for (int d = 0; d < N::kDims; ++d) *reinterpret_cast<f32x4*>(ow + 16 * d) = o[n][d];
      __syncthreads();
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
      if (!cut) {
        finish(r, x, m, l);
        continue;
      }
#pragma unroll
      for (int i = 0; i < kPer; i += 4)
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4{__float_as_uint(x[i]), __float_as_uint(x[i + 1]), __float_as_uint(x[i + 2]), __float_as_uint(x[i + 3])},
            mres, 4 * (r * D + od + i), 0, kSc1);
      if ((tid & 15) == 0) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(m), mres, 4 * (N::kRows * D + r), 0, kSc1);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l), mres, 4 * (N::kRows * (D + 1) + r), 0, kSc1);
      }
    }
    if (cut) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (each wave's stores have completed)
    __syncthreads();  // the waves' V rows are free again
    if (cut) {
      if (tid == 0)
        last = __hip_atomic_fetch_add(tickets + pp.first, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               (unsigned)(pp.count - 1);
      __syncthreads();
      if (last) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const int r = 16 * n + orow;
          if (r >= rows) break;
          float m = -INFINITY, l = 0.0f, x[kPer] = {};
          constexpr int kBatch = 4;
          for (int k0 = 0; k0 < pp.count; k0 += kBatch) {
            float pm[kBatch], pl[kBatch];
            u32x4 px[kBatch][kPer / 4];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              const int wk = pp.first + min(k0 + k, pp.count - 1);
              const __amdgpu_buffer_rsrc_t res =
                  rsrc(parts + (int64_t)plan_slot(run.place.start, wk, run.per) * N::kPart, N::kPart * 4);
              pm[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(res, 4 * (N::kRows * D + r), 0, kSc1));
              pl[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(res, 4 * (N::kRows * (D + 1) + r), 0, kSc1));
#pragma unroll
              for (int i = 0; i < kPer / 4; ++i)
                px[k][i] = __builtin_amdgcn_raw_buffer_load_b128(res, 4 * (r * D + od + 4 * i), 0, kSc1);
            }
            float m_new = m;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) m_new = fmaxf(m_new, pm[k]);
            const float f0 = __builtin_amdgcn_exp2f(m - finite_max(m_new));
            l *= f0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) x[i] *= f0;
            m = m_new;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              if (k0 + k >= pp.count) break;
              const float f = __builtin_amdgcn_exp2f(pm[k] - finite_max(m));
              l = fmaf(pl[k], f, l);
#pragma unroll
              for (int i = 0; i < kPer; ++i) x[i] = fmaf(__uint_as_float(px[k][i / 4][i % 4]), f, x[i]);
            }
          }
          finish(r, x, m, l);
        }
        if (tid == 0) __hip_atomic_store(tickets + pp.first, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    run.unit += take;
    if (run.unit < run.end) plan_next(a, shape, run, units);
  }
}

// Partial results and tickets of the largest launch fit the workspace.
constexpr int kNarrowGroups[3] = {768, 512, 256};  // NQ 1, 2, 4: what the GPU holds at once
template <int NQ, int GROUPS>
constexpr bool fits() {
  return GROUPS <= kPagedTicketWords && GROUPS % 8 == 0 &&
         4ll * kPagedTicketWords + 2ll * GROUPS * Narrow<128, false, NQ>::kPart * 4 <= HK_PAGED_WORKSPACE;
}
static_assert(fits<1, kNarrowGroups[0]>() && fits<2, kNarrowGroups[1]>() && fits<4, kNarrowGroups[2]>(), "workspace");

template <int D, bool E4M3>
void launch(const PagedAttnArgs& a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.max_new * a.group;
  if (rows <= 16)
    hipLaunchKernelGGL((paged_narrow_kernel<D, E4M3, 1>), dim3(kNarrowGroups[0]), dim3(kThreads), 0, stream, a);
  else if (rows <= 32)
    hipLaunchKernelGGL((paged_narrow_kernel<D, E4M3, 2>), dim3(kNarrowGroups[1]), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_narrow_kernel<D, E4M3, 4>), dim3(kNarrowGroups[2]), dim3(kThreads), 0, stream, a);
}

}  // namespace

int launch_paged_attention(const PagedAttnArgs& a, int head_dim, hipStream_t stream) {
  const bool e4m3 = a.c.elt == 1;
  if (head_dim == 64)
    e4m3 ? launch<64, true>(a, stream) : launch<64, false>(a, stream);
  else
    e4m3 ? launch<128, true>(a, stream) : launch<128, false>(a, stream);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : hip_fail(err, "paged attention launch");
}

}  // namespace hk
