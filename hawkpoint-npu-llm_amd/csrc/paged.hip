// The paged KV cache's entry points (include/hk_paged.h) and the kernels of
// its append, fork and compaction.  The attention is in paged_attention.hip.
#include <cmath>
#include <initializer_list>
#include <string>

#include "hk.h"
#include "hk_common.h"
#include "hk_internal.h"
#include "paged.h"

namespace hk {
namespace {

constexpr int kWords = HK_PAGED_WORKSPACE / 4;  // int32 words of a workspace

// ---- append ----

struct AppendArgs {
  PagedPool c;
  PagedBatch b;
  const uint16_t* qkv;
  uint16_t* q_out;
  const float* cos_tab;
  const float* sin_tab;
  const int32_t* status;  // optional: nothing is done unless its first word is HK_PAGED_DONE
  int64_t qkv_stride, q_stride;
  int q_heads;
};

// x / scale as e4m3: saturated, NaN stays NaN (v_cvt_pk_fp8_f32 rounds to
// nearest even; its own result for values past the largest is not used).
__device__ __forceinline__ float saturated(float x, float scale) {
  const float y = x / scale;
  return y != y ? y : fminf(fmaxf(y, -448.0f), 448.0f);
}
__device__ __forceinline__ u32x2_t e4m3x8(const float (&x)[8], float scale) {
  u32x2_t o;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(saturated(x[4 * w], scale), saturated(x[4 * w + 1], scale), 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(saturated(x[4 * w + 2], scale), saturated(x[4 * w + 3], scale), v, true);
    o[w] = v;
  }
  return o;
}

__device__ __forceinline__ void unpack8(const u32x4& v, float (&x)[8]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    x[2 * w] = bf_lo(v[w]);
    x[2 * w + 1] = bf_hi(v[w]);
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]), f32x2_to_bf16x2(x[4], x[5]),
               f32x2_to_bf16x2(x[6], x[7])};
}

// Eight values at dimension d of a pool row.
template <bool E4M3>
__device__ __forceinline__ void store8(char* row, int d, const float (&x)[8], float scale) {
  if constexpr (E4M3)
    stg(reinterpret_cast<u32x2_t*>(row + d), e4m3x8(x, scale));
  else
    stg(reinterpret_cast<u32x4*>(row + 2 * d), pack8(x));
}

// One workgroup per token.  A thread takes 8 dimensions of a head's first half
// and the 8 they turn with, 16 bytes each; the work items of a token are the q
// heads, the k heads and the v heads times D / 16: 384 for 8 k and 32 q heads of
// 128, a round and a half of the workgroup, 72 for 14 and 2 of 64.  It finds the
// token's entry by going through all of `first`, one load a thread up to 256
// entries: nothing has to be planned before.  Many tokens are bound by memory:
// pieces of 5 prompts (3205 rows, e4m3) in 14.8 us, 5.0 TB/s read and written, in
// bf16 14.2 us and 5.6 TB/s (a large copy reaches 4.7); of 14 heads on 2 of 64,
// where a workgroup has 5 KB to move, in 5.7 us and 2.7 TB/s.  A decode step's 61
// rows are bound by the launch and four loads that wait for each other (entry,
// length, page, row): 4.6 to 5.5 us a call, 3.0 to 3.5 of them the kernel.
template <int D, bool E4M3>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  constexpr int kItems = D / 16;
  __shared__ int found;
  const int tok = blockIdx.x;
  if (threadIdx.x == 0) found = -1;
  __syncthreads();
  for (int e = threadIdx.x; e < a.b.n; e += 256) {
    const int2 r = entry_rows(a.b, e);
    if (tok >= r.x && tok < r.y) found = e;
  }
  __syncthreads();
  if (found < 0) return;
  if (a.status && *a.status != HK_PAGED_DONE) return;  // (in front of the search it costs calls without one 0.1 to 0.3 us)
  const int2 r = entry_rows(a.b, found), s = entry_seq(a.c, a.b, found);
  const int p = s.y - r.y + tok;
  if (p < 0) return;
  const int page = ldg(a.c.table + (int64_t)s.x * a.c.width + (p >> a.c.page_shift));
  const bool there = (unsigned)page < (unsigned)a.c.pages;
  const int64_t base = page * a.c.page_bytes;
  const int slot = p & ((1 << a.c.page_shift) - 1);
  const uint16_t* in = a.qkv + tok * a.qkv_stride;
  const int heads = a.q_heads + 2 * a.c.kv_heads;
  for (int i = threadIdx.x; i < heads * kItems; i += 256) {
    const int h = i / kItems, d = 8 * (i % kItems), g = h - a.q_heads;
    const u32x4 lo = load16(in + h * D + d), hi = load16(in + h * D + D / 2 + d);
    float x[8], y[8];
    unpack8(lo, x);
    unpack8(hi, y);
    if (g < a.c.kv_heads && a.cos_tab) {
      const float* cs = a.cos_tab + (int64_t)p * (D / 2) + d;
      const float* sn = a.sin_tab + (int64_t)p * (D / 2) + d;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float c1 = ldg(cs + q), s1 = ldg(sn + q), u = x[q], w = y[q];
        x[q] = u * c1 - w * s1;
        y[q] = w * c1 + u * s1;
      }
    }
    if (g < 0) {
      if (a.q_out) {
        uint16_t* o = a.q_out + tok * a.q_stride + h * D;
        stg(reinterpret_cast<u32x4*>(o + d), pack8(x));
        stg(reinterpret_cast<u32x4*>(o + D / 2 + d), pack8(y));
      }
    } else if (there) {
      const bool key = g < a.c.kv_heads;
      const int kh = key ? g : g - a.c.kv_heads;
      const float scale = E4M3 ? (key ? a.c.k_scale : a.c.v_scale)[kh] : 1.0f;
      char* row = (key ? a.c.k : a.c.v) + base + (((int64_t)kh << a.c.page_shift) + slot) * D * a.c.elt;
      store8<E4M3>(row, d, x, scale);
      store8<E4M3>(row, D / 2 + d, y, scale);
    }
  }
}

// ---- moving slots between pages ----

// A move: the first `slots` slots of page `from` to page `to`, every layer,
// keys and values.
struct Move {
  int from, to, slots;
};

struct MoveArgs {
  char* k;
  char* v;
  const Move* moves;
  const int* count;
  int64_t layer_bytes, page_bytes;
  int layers, kv_heads, page_shift, row_bytes;
  int whole;  // every move is of whole pages, whose heads are one run
  // compaction: the tables' cells, and the new numbers of the pages from `live` on
  const int32_t* table;
  int32_t* table_out;
  const int32_t* live;
  const int* place;
  int64_t cells;
  int pages;
};

// Pieces of 16 KiB of the runs (move, layer, keys or values, head) go round the
// workgroups; before that the tables get the pages' new numbers, where there
// are any.  What bounds it is memory: 475 pages of 2 MB moved in 399 us (5.0
// TB/s read and written, a large copy reaches 4.7), a prompt's page copied to 8
// answers at 6.0.  The stores stream, as nobody reads the copies soon (134 us
// for 192 answers against 156); the loads do not, as a page may be the source of
// several copies (streaming loads too: 172; without several copies 402 and 406).
constexpr int kPieceLoads = 4;
constexpr int kPieceBytes = 256 * 16 * kPieceLoads;
__global__ __launch_bounds__(256) void paged_move_kernel(MoveArgs a) {
  const int heads = a.whole ? 1 : a.kv_heads, per_move = a.layers * 2 * heads;
  const int64_t head_bytes = (int64_t)a.row_bytes << a.page_shift, most = a.whole ? head_bytes * a.kv_heads : head_bytes;
  const int pieces = (int)((most + kPieceBytes - 1) / kPieceBytes);
  if (a.cells) {
    const int first = *a.live;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.cells; i += (int64_t)gridDim.x * 256) {
      const int p = a.table[i];
      a.table_out[i] = p >= first && p < a.pages ? a.place[p] : p;
    }
  }
  const int64_t all = (int64_t)*a.count * per_move * pieces;
  for (int64_t i = blockIdx.x; i < all; i += gridDim.x) {
    const int64_t run = i / pieces;
    const Move m = a.moves[run / per_move];
    const int r = (int)(run % per_move), h = r % heads, kv = r / heads % 2, layer = r / heads / 2;
    char* pool = (kv ? a.v : a.k) + layer * a.layer_bytes + h * head_bytes;
    const int64_t at = (i - run * pieces) * kPieceBytes + threadIdx.x * 16;
    const int64_t bytes = (a.whole ? most : (int64_t)m.slots * a.row_bytes) - at;
    const char* src = pool + m.from * a.page_bytes + at;
    char* dst = pool + m.to * a.page_bytes + at;
    u32x4 x[kPieceLoads];
#pragma unroll
    for (int k = 0; k < kPieceLoads; ++k)
      if (k * 4096 < bytes) x[k] = load16(src + k * 4096);
#pragma unroll
    for (int k = 0; k < kPieceLoads; ++k)
      if (k * 4096 < bytes) __builtin_nontemporal_store(x[k], (__attribute__((address_space(1))) u32x4*)(dst + k * 4096));
  }
}

// ---- bookkeeping: one workgroup, so that a barrier orders its steps ----

constexpr int kBook = 1024;
constexpr int kBookWaves = kBook / 64;

// Words that other threads of the workgroup change with atomics, or that are
// read back in another order than written.
__device__ __forceinline__ int peek(const int* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void poke(int* p, int v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void bump(int* p, int by) {
  __hip_atomic_fetch_add(p, by, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Barrier after which every thread sees what the others stored before it.
__device__ __forceinline__ void book_sync() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Exclusive prefix sum of v over the workgroup, and the total.
__device__ __forceinline__ int book_scan(int v, int* wave_sums, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int u = __shfl_up(s, m, 64);
    if (lane >= m) s += u;
  }
  __syncthreads();  // (the sums of an earlier scan have been read)
  if (lane == 63) wave_sums[wave] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kBookWaves; ++w) {
    const int u = wave_sums[w];
    if (w < wave) before += u;
    all += u;
  }
  total = all;
  return before + s - v;
}

// This wave's run of the pages [from, to): whole groups of 64.
__device__ __forceinline__ int2 wave_pages(int from, int to) {
  const int groups = (to - from + 63) / 64, per = (groups + kBookWaves - 1) / kBookWaves;
  const int lo = from + (threadIdx.x >> 6) * per * 64;
  return make_int2(min(lo, to), min(lo + per * 64, to));
}

// Counts the pages of [from, to) whose refs are positive (or not, for FREE),
// per wave and in all.
template <bool FREE>
__device__ __forceinline__ int book_count(const int* refs, int from, int to, int* wave_sums, int& before) {
  const int2 w = wave_pages(from, to);
  int n = 0;
  for (int p = w.x + (threadIdx.x & 63); p < w.y; p += 64) n += (peek(refs + p) > 0) != FREE;
  int total;
  const int mine = book_scan(n, wave_sums, total);
  before = __builtin_amdgcn_readfirstlane(mine);  // pages in the waves before this one
  return total;
}

// take(rank, page) for those pages in ascending order, ranks below `most`.
template <bool FREE, typename F>
__device__ __forceinline__ void book_list(const int* refs, int from, int to, int before, int most, F take) {
  const int2 w = wave_pages(from, to);
  const int lane = threadIdx.x & 63;
  for (int p0 = w.x; p0 < w.y && before < most; p0 += 64) {
    const int p = p0 + lane;
    const bool is = p < w.y && (peek(refs + p) > 0) != FREE;
    const unsigned long long mask = __ballot(is);
    const int rank = before + __popcll(mask & ((1ull << lane) - 1));
    if (is && rank < most) take(rank, p);
    before += __popcll(mask);
  }
}

// ---- fork ----

struct ForkArgs {
  int32_t* table;
  int32_t* length;
  int32_t* refs;
  const int32_t* child;
  const int32_t* parent;
  const int32_t* keep;
  const int32_t* grow;
  int32_t* status;
  int n, pages, seqs, width, page_shift;
  // workspace: the entries as read, and what they get
  int* entry;    // [7][n] (LDS false)
  int* owner;    // [seqs] first entry of a child
  int* claim;    // [pages] first entry that wants a page
  int* fresh;    // [pages] free pages in order
  int* rows;     // [n, width] the parents' rows
  Move* moves;   // [n]
  int* count;    // moves
};

// The pages' counts without the children's rows and with what they share say
// what is free; a prefix sum over the entries' needs and one over the free pages
// pair the two up, and only then anything is written.  One workgroup does it
// all, as its steps wait for each other and a barrier is cheaper than a launch
// (4 us).  What it takes is round trips to memory, one after the other (about a
// microsecond each, ten of them; 64 sequences, one more token each: 11 us in a
// pool of 2000 pages).  The pool's counts are gone through in every call, sixteen
// waves 64 pages at a time: with 20 000 pages the step takes 13 to 16 us (the
// copy's launch included), with 200 000 32 to 39, whether or not a page is needed.
// So
// the rows of all entries are gone through together, a thread per (entry,
// column): 192 answers to 24 prompts in 17 us, where a wave per entry took 68.
// Up to kForkLds entries are kept in LDS, more in the workspace.
constexpr int kForkLds = 1024;
template <bool LDS>
__global__ __launch_bounds__(kBook) void paged_fork_kernel(ForkArgs a) {
  __shared__ int sums[kBookWaves];
  __shared__ int bad, moved, longest;
  __shared__ int entry_lds[LDS ? 7 * kForkLds : 1];
  const int tid = threadIdx.x, n = a.n, shift = a.page_shift, stride = LDS ? kForkLds : n;
  int* const child = LDS ? entry_lds : a.entry;
  int* const parent = child + stride;
  int* const keep = parent + stride;
  int* const total = keep + stride;  // pages
  int* const start = total + stride; // first of its new pages
  int* const want = start + stride;  // the partly filled page; ~page - 1: taken over; -1: none
  int* const held = want + stride;   // pages before the call
  const int slots = a.width << shift, mask = (1 << shift) - 1;
  auto length = [&](int s) { return min(max(a.length[s], 0), slots); };
  if (tid == 0) {
    bad = n;
    moved = 0;
    longest = 1;
  }
  for (int i = tid; i < n; i += kBook) {
    const int c = a.child ? a.child[i] : i;
    if ((unsigned)c < (unsigned)a.seqs) poke(a.owner + c, n);
  }
  book_sync();
  // read and check the entries
  int mine = n;
  for (int i = tid; i < n; i += kBook) {
    const int c = a.child ? a.child[i] : i, q = a.parent ? a.parent[i] : c;
    const bool has = (unsigned)q < (unsigned)a.seqs;
    const int64_t most = has ? length(q) : 0, k = a.keep ? a.keep[i] : most, g = a.grow ? a.grow[i] : 0;
    bool ok = (unsigned)c < (unsigned)a.seqs && k >= 0 && k <= most && g >= 0 && k + g <= slots;
    int w = -1;
    if (ok) {
      __hip_atomic_fetch_min(a.owner + c, i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int t = (int)((k + g + mask) >> shift), h = (length(c) + mask) >> shift;
      child[i] = c;
      parent[i] = has ? q : c;
      keep[i] = (int)k;
      total[i] = t;
      held[i] = h;
      atomicMax(&longest, max(t, h) - (!has || q == c ? (int)(k >> shift) : 0));
      if (k & mask) {
        w = a.table[(int64_t)q * a.width + (k >> shift)];
        ok = (unsigned)w < (unsigned)a.pages;
        if (ok) poke(a.claim + w, n);
      }
    }
    want[i] = w;
    if (!ok) mine = min(mine, i);
  }
  book_sync();
  for (int i = tid; i < n; i += kBook) {
    if (i >= mine) break;
    if (peek(a.owner + child[i]) != i) mine = min(mine, i);
  }
  if (mine < n) atomicMin(&bad, mine);
  __syncthreads();
  if (bad < n) {
    if (tid == 0) {
      *a.count = 0;
      a.status[0] = HK_PAGED_BAD_ENTRY, a.status[1] = bad;
    }
    return;
  }
  // f(entry, column) for every entry and the columns that the call concerns: an
  // entry that goes on from itself keeps its full pages without a look
  int columns = 0;
  while ((1 << columns) < longest) ++columns;
  auto cells = [&](auto f) {
    const int64_t all = (int64_t)n << columns;
    for (int64_t x = tid; x < all; x += kBook) {
      const int i = (int)(x >> columns), j = (int)(x & ((1 << columns) - 1)) + (child[i] == parent[i] ? keep[i] >> shift : 0);
      f(i, j);
    }
  };
  // the counts without what the children held and with what they share (by 1);
  // the same taken back (by -1)
  auto share = [&](int by) {
    cells([&](int i, int j) {
      const int full = keep[i] >> shift;
      if (j < held[i]) {
        const int p = a.table[(int64_t)child[i] * a.width + j];
        if ((unsigned)p < (unsigned)a.pages) bump(a.refs + p, -by);
      }
      if (j < full) {  // (never of the sequence itself)
        const int p = a.table[(int64_t)parent[i] * a.width + j];
        if ((unsigned)p < (unsigned)a.pages) bump(a.refs + p, by);
        a.rows[(int64_t)i * a.width + j] = p;
      }
    });
  };
  share(1);
  for (int i = tid; i < n; i += kBook)
    if (want[i] >= 0) __hip_atomic_fetch_min(a.claim + want[i], i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  book_sync();
  // a wanted page that nobody keeps now goes to its first claimant
  int need = 0;
  const int per = (n + kBook - 1) / kBook;  // consecutive entries per thread, for the prefix sum
  const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
  for (int i = i0; i < i1; ++i) {
    bool taken = false;
    if (want[i] >= 0) taken = peek(a.refs + want[i]) <= 0 && peek(a.claim + want[i]) == i;
    if (taken) want[i] = ~want[i] - 1;
    need += total[i] - (keep[i] >> shift) - (taken ? 1 : 0);
  }
  int all, before;
  const int offset = book_scan(need, sums, all);  // (its barriers come before the counts change)
  for (int i = i0, at = offset; i < i1; ++i) {
    if (want[i] < -1) poke(a.refs + ~(want[i] + 1), 1);
    start[i] = at;
    at += total[i] - (keep[i] >> shift) - (want[i] < -1 ? 1 : 0);
  }
  book_sync();
  const int free_pages = book_count<true>(a.refs, 0, a.pages, sums, before);
  if (free_pages < all) {
    for (int i = i0; i < i1; ++i)
      if (want[i] < -1) poke(a.refs + ~(want[i] + 1), 0);
    book_sync();
    share(-1);
    if (tid == 0) {
      *a.count = 0;
      a.status[0] = HK_PAGED_FULL, a.status[1] = all - free_pages;
    }
    return;
  }
  book_list<true>(a.refs, 0, a.pages, before, all, [&](int rank, int page) { a.fresh[rank] = page; });
  book_sync();
  for (int r = tid; r < all; r += kBook) poke(a.refs + a.fresh[r], 1);
  // the rows, the copies and the lengths
  cells([&](int i, int j) {
    const int full = keep[i] >> shift, taken = want[i] < -1;
    int p;
    if (j < full)
      p = a.rows[(int64_t)i * a.width + j];
    else if (j < full + taken)
      p = ~(want[i] + 1);
    else if (j < total[i])
      p = a.fresh[start[i] + j - full - taken];
    else if (j < held[i])
      p = -1;
    else
      return;
    a.table[(int64_t)child[i] * a.width + j] = p;
  });
  for (int i = tid; i < n; i += kBook)
    if (want[i] >= 0) a.moves[atomicAdd(&moved, 1)] = Move{want[i], a.fresh[start[i]], keep[i] & mask};
  book_sync();
  for (int i = tid; i < n; i += kBook) start[i] = keep[i] + (a.grow ? a.grow[i] : 0);
  book_sync();  // (grow may be the lengths)
  for (int i = tid; i < n; i += kBook) a.length[child[i]] = start[i];
  if (tid == 0) {
    *a.count = moved;
    a.status[0] = HK_PAGED_DONE, a.status[1] = 0;
  }
}

// ---- compaction ----

struct CompactArgs {
  const int32_t* refs;
  int32_t* refs_out;
  int32_t* live;
  int pages;
  int* place;   // [pages] new number of each page from L on
  Move* moves;  // [pages / 2]
  int* count;
};

// With L live pages there are as many free ones below L as live ones from L on:
// the pairs come from counting both, a wave 64 pages at a time (__ballot), in
// order, and the moves touch nothing twice.  One workgroup; 512 pages take 4.2
// us, 1900 take 6.6, beside 9 and 392 for the moves.
__global__ __launch_bounds__(kBook) void paged_compact_kernel(CompactArgs a) {
  __shared__ int sums[kBookWaves];
  const int tid = threadIdx.x;
  int before, holes, movers;
  const int live = book_count<false>(a.refs, 0, a.pages, sums, before);
  holes = book_count<true>(a.refs, 0, live, sums, before);
  book_list<true>(a.refs, 0, live, before, holes, [&](int rank, int page) { a.moves[rank].to = page; });
  movers = book_count<false>(a.refs, live, a.pages, sums, before);  // as many as holes
  book_list<false>(a.refs, live, a.pages, before, movers, [&](int rank, int page) { a.moves[rank].from = page; });
  // (an entry that names a page without references keeps its number)
  for (int p = live + tid; p < a.pages; p += kBook) a.place[p] = p;
  book_sync();
  for (int i = tid; i < movers; i += kBook) {
    const Move m = a.moves[i];
    a.place[m.from] = m.to;
    a.moves[i].slots = a.refs[m.from];  // whole pages move: the word carries the count to its new place
  }
  if (a.refs_out != a.refs)
    for (int p = tid; p < live; p += kBook) a.refs_out[p] = a.refs[p];
  book_sync();
  for (int i = tid; i < movers; i += kBook) a.refs_out[a.moves[i].to] = a.moves[i].slots;
  for (int p = live + tid; p < a.pages; p += kBook) a.refs_out[p] = 0;
  if (tid == 0) *a.live = live, *a.count = movers;
}

// ---- checks ----

// Arrays of 32-bit words.  Scalar loads leave an address's last two bits out
// where vector loads do not, so a kernel would read two batches from one
// misaligned array and go by both.
int check_words(const char* who, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if ((uintptr_t)p % 4) return fail(std::string(who) + ": int32 and float32 arrays must be aligned to 4 bytes");
  return 0;
}

int check_cache(const char* who, const hk_paged_cache* c) {
  const std::string at = std::string(who) + ": ";
  if (!c) return fail(at + "null cache");
  if (!c->k || !c->v || !c->table || !c->length || !c->refs) return fail(at + "null pointer in the cache");
  if (c->dtype != HK_PAGED_BF16 && c->dtype != HK_PAGED_E4M3) return fail(at + "unknown dtype");
  if (c->head_dim != 64 && c->head_dim != 128) {
    set_error(at + "only head_dim 64 and 128 are supported");
    return HK_ERR_UNSUPPORTED;
  }
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) {
    set_error(at + "page_size must be 16, 32, 64, 128 or 256");
    return HK_ERR_UNSUPPORTED;
  }
  if (c->layers <= 0 || c->kv_heads <= 0 || c->pages <= 0 || c->seqs <= 0 || c->table_width <= 0)
    return fail(at + "layers, kv_heads, pages, seqs and table_width must be positive");
  if (c->kv_heads > 1024) return fail(at + "more than 1024 kv heads");
  if ((int64_t)c->table_width * c->page_size > INT32_MAX / 2) return fail(at + "more than 2^30 slots per sequence");
  const int64_t page = (int64_t)c->kv_heads * c->page_size * c->head_dim, unit = c->dtype == HK_PAGED_BF16 ? 8 : 16;
  if (c->page_stride < page || c->page_stride % unit) return fail(at + "page_stride below a page or not of 16 bytes");
  if (c->layers > 1 && (c->layer_stride < page || c->layer_stride % unit))
    return fail(at + "layer_stride below a page or not of 16 bytes");
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16) return fail(at + "pools must be aligned to 16 bytes");
  if (c->dtype == HK_PAGED_E4M3 && (!c->k_scale || !c->v_scale)) return fail(at + "e4m3 needs k_scale and v_scale");
  return check_words(who, {c->table, c->length, c->refs, c->k_scale, c->v_scale, c->status});
}

int check_batch(const char* who, const hk_paged_cache* c, int32_t layer, const int32_t* seqs, const int32_t* first,
                int32_t n, int32_t tokens, int32_t q_heads) {
  const std::string at = std::string(who) + ": ";
  if (layer < 0 || layer >= c->layers) return fail(at + "layer outside the cache");
  if (!first) return fail(at + "null pointer");
  if (n < 0 || tokens < 0) return fail(at + "negative batch");
  if (n > HK_PAGED_MAX_BATCH) return fail(at + "more than 4096 sequences in a call");
  if (q_heads <= 0 || q_heads % c->kv_heads != 0) return fail(at + "q_heads must be a positive multiple of kv_heads");
  if (q_heads > 4096) return fail(at + "more than 4096 q heads");
  return check_words(who, {seqs, first});
}

int check_rows(const char* who, const char* name, const void* p, int64_t stride, int64_t width) {
  if ((uintptr_t)p % 16 || stride % 8) return fail(std::string(who) + ": " + name + " must be aligned to 16 bytes");
  if (stride < width) return fail(std::string(who) + ": " + name + "'s stride is below its width");
  return 0;
}

int check_workspace(const char* who, const void* p) {
  if (!p) return fail(std::string(who) + ": null workspace");
  if ((uintptr_t)p % 256) return fail(std::string(who) + ": the workspace must be aligned to 256 bytes");
  return 0;
}

int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

PagedPool pool_of(const hk_paged_cache* c, int32_t layer) {
  PagedPool p = {};
  p.elt = c->dtype == HK_PAGED_BF16 ? 2 : 1;
  const int64_t at = (int64_t)layer * c->layer_stride * p.elt;
  p.k = static_cast<char*>(c->k) + at;
  p.v = static_cast<char*>(c->v) + at;
  if (c->dtype == HK_PAGED_E4M3) {
    p.k_scale = c->k_scale + (int64_t)layer * c->kv_heads;
    p.v_scale = c->v_scale + (int64_t)layer * c->kv_heads;
  }
  p.table = c->table;
  p.length = c->length;
  p.page_bytes = c->page_stride * p.elt;
  p.kv_heads = c->kv_heads;
  p.page_shift = log2_of(c->page_size);
  p.pages = c->pages;
  p.seqs = c->seqs;
  p.width = c->table_width;
  return p;
}

MoveArgs moves_of(const hk_paged_cache* c, const Move* moves, const int* count, bool whole) {
  MoveArgs m = {};
  const int elt = c->dtype == HK_PAGED_BF16 ? 2 : 1;
  m.k = static_cast<char*>(c->k);
  m.v = static_cast<char*>(c->v);
  m.moves = moves;
  m.count = count;
  m.layer_bytes = c->layer_stride * elt;
  m.page_bytes = c->page_stride * elt;
  m.layers = c->layers;
  m.kv_heads = c->kv_heads;
  m.page_shift = log2_of(c->page_size);
  m.row_bytes = c->head_dim * elt;
  m.whole = whole;
  return m;
}

// Eight workgroups per CU: 16 KiB in flight each.  Four take 15.7 us instead of
// 14.9 for the 512-page pool and 136 instead of 133 for 192 answers, sixteen
// 13.4 instead of 12.8 for a step that copies nothing.
constexpr int kMoveGroups = 2048;

#define HK_TRY(call)            \
  do {                          \
    const int rc_ = (call);     \
    if (rc_ != HK_OK) return rc_; \
  } while (0)

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

int hk_paged_append(const hk_paged_cache* cache, int32_t layer, const uint16_t* qkv, int64_t qkv_stride,
                    const float* rope_cos, const float* rope_sin, int32_t positions, const int32_t* seqs,
                    const int32_t* first, int32_t n, int32_t tokens, int32_t q_heads, uint16_t* q_out,
                    int64_t q_out_stride, void* stream) {
  static const char who[] = "hk_paged_append";
  HK_TRY(check_cache(who, cache));
  HK_TRY(check_batch(who, cache, layer, seqs, first, n, tokens, q_heads));
  if (!qkv) return fail("hk_paged_append: null pointer");
  const int d = cache->head_dim;
  HK_TRY(check_rows(who, "qkv", qkv, qkv_stride, (int64_t)(q_heads + 2 * cache->kv_heads) * d));
  if (q_out) HK_TRY(check_rows(who, "q_out", q_out, q_out_stride, (int64_t)q_heads * d));
  if (q_out == qkv && q_out_stride != qkv_stride) return fail("hk_paged_append: in place only with equal strides");
  if (!rope_cos != !rope_sin) return fail("hk_paged_append: give both RoPE tables or neither");
  if (rope_cos && ((uintptr_t)rope_cos | (uintptr_t)rope_sin) % 16)
    return fail("hk_paged_append: the RoPE tables must be aligned to 16 bytes");
  if (rope_cos && positions < (int64_t)cache->table_width * cache->page_size)
    return fail("hk_paged_append: RoPE tables shorter than the longest sequence");
  if (tokens >= 1 << 24) {  // (a launch has 2^32 threads at most)
    set_error("hk_paged_append: 2^24 tokens or more in a call");
    return HK_ERR_UNSUPPORTED;
  }
  if (n == 0 || tokens == 0) return 0;
  AppendArgs a = {pool_of(cache, layer), {seqs, first, n, tokens}, qkv, q_out, rope_cos, rope_sin,
                  cache->status, qkv_stride, q_out_stride, q_heads};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool e4m3 = cache->dtype == HK_PAGED_E4M3;
  const auto kernel = d == 64 ? (e4m3 ? paged_append_kernel<64, true> : paged_append_kernel<64, false>)
                              : (e4m3 ? paged_append_kernel<128, true> : paged_append_kernel<128, false>);
  return paged_launch("paged append launch", kernel, tokens, 256, st, a);
}

int hk_paged_attention(const hk_paged_cache* cache, int32_t layer, const uint16_t* q, int64_t q_stride,
                       const int32_t* seqs, const int32_t* first, int32_t n, int32_t tokens, int32_t max_new,
                       int32_t q_heads, float scale, int32_t window, uint16_t* out, int64_t out_stride, float* lse,
                       void* workspace, void* stream) {
  static const char who[] = "hk_paged_attention";
  HK_TRY(check_cache(who, cache));
  HK_TRY(check_batch(who, cache, layer, seqs, first, n, tokens, q_heads));
  if (!q || !out) return fail("hk_paged_attention: null pointer");
  const int64_t width = (int64_t)q_heads * cache->head_dim;
  HK_TRY(check_rows(who, "q", q, q_stride, width));
  HK_TRY(check_rows(who, "out", out, out_stride, width));
  HK_TRY(check_workspace(who, workspace));
  HK_TRY(check_words(who, {lse}));
  if (max_new < 1) return fail("hk_paged_attention: max_new must be positive");
  if ((int64_t)tokens * q_heads > INT32_MAX / 2) {
    set_error("hk_paged_attention: more than 2^30 rows (tokens x q_heads)");
    return HK_ERR_UNSUPPORTED;
  }
  if (out == q && out_stride != q_stride) return fail("hk_paged_attention: in place only with equal strides");
  if (window < 0) return fail("hk_paged_attention: negative window");
  if (!std::isfinite(scale) || !(scale > 0.0f)) return fail("hk_paged_attention: scale must be finite and positive");
  if (n == 0 || tokens == 0) return 0;
  PagedAttnArgs a = {};
  a.c = pool_of(cache, layer);
  a.b = {seqs, first, n, tokens};
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.q_heads = q_heads;
  a.group = q_heads / cache->kv_heads;
  a.window = window;
  a.max_new = max_new;
  a.scale = scale;
  a.workspace = workspace;
  return launch_paged_attention(a, cache->head_dim, static_cast<hipStream_t>(stream));
}

int hk_paged_fork(const hk_paged_cache* cache, const int32_t* child, const int32_t* parent, const int32_t* keep,
                  const int32_t* grow, int32_t n, int32_t* status, void* workspace, void* stream) {
  static const char who[] = "hk_paged_fork";
  HK_TRY(check_cache(who, cache));
  if (!status) return fail("hk_paged_fork: null status");
  HK_TRY(check_workspace(who, workspace));
  HK_TRY(check_words(who, {child, parent, keep, grow, status}));
  if (n < 1 || n > cache->seqs) return fail("hk_paged_fork: n outside 1 .. seqs");
  ForkArgs a = {};
  a.table = cache->table;
  a.length = cache->length;
  a.refs = cache->refs;
  a.child = child;
  a.parent = parent;
  a.keep = keep;
  a.grow = grow;
  a.status = status;
  a.n = n;
  a.pages = cache->pages;
  a.seqs = cache->seqs;
  a.width = cache->table_width;
  a.page_shift = log2_of(cache->page_size);
  // the workspace's first words stay the attention's (zero between calls)
  const int64_t words = kPagedTicketWords + 64 + 10 * (int64_t)n + a.seqs + 2 * (int64_t)a.pages + (int64_t)n * a.width;
  if (words > kWords) {
    set_error("hk_paged_fork: entries, tables and pages beyond the workspace");
    return HK_ERR_UNSUPPORTED;
  }
  int* w = static_cast<int*>(workspace) + kPagedTicketWords;
  a.count = w;
  a.entry = w + 64;
  a.owner = a.entry + 7 * (int64_t)n;
  a.claim = a.owner + a.seqs;
  a.fresh = a.claim + a.pages;
  a.rows = a.fresh + a.pages;
  a.moves = reinterpret_cast<Move*>(a.rows + (int64_t)n * a.width);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  HK_TRY(paged_launch("paged fork launch", n <= kForkLds ? paged_fork_kernel<true> : paged_fork_kernel<false>, 1, kBook, st, a));
  return paged_launch("paged fork copy launch", paged_move_kernel, kMoveGroups, 256, st,
                      moves_of(cache, a.moves, a.count, false));
}

int hk_paged_compact(const hk_paged_cache* cache, int32_t* table_out, int32_t* refs_out, int32_t* live_out,
                     void* workspace, void* stream) {
  static const char who[] = "hk_paged_compact";
  HK_TRY(check_cache(who, cache));
  if (!table_out || !refs_out || !live_out) return fail("hk_paged_compact: null pointer");
  HK_TRY(check_workspace(who, workspace));
  HK_TRY(check_words(who, {table_out, refs_out, live_out}));
  CompactArgs a = {};
  a.refs = cache->refs;
  a.refs_out = refs_out;
  a.live = live_out;
  a.pages = cache->pages;
  const int64_t words = kPagedTicketWords + 64 + (int64_t)a.pages + 3 * ((int64_t)a.pages / 2 + 1);
  if (words > kWords) {
    set_error("hk_paged_compact: pages beyond the workspace");
    return HK_ERR_UNSUPPORTED;
  }
  int* w = static_cast<int*>(workspace) + kPagedTicketWords;
  a.count = w;
  a.place = w + 64;
  a.moves = reinterpret_cast<Move*>(a.place + a.pages);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  HK_TRY(paged_launch("paged compact launch", paged_compact_kernel, 1, kBook, st, a));
  MoveArgs m = moves_of(cache, a.moves, a.count, true);
  m.table = cache->table;
  m.table_out = table_out;
  m.live = live_out;
  m.place = a.place;
  m.cells = (int64_t)cache->seqs * cache->table_width;
  m.pages = a.pages;
  return paged_launch("paged move launch", paged_move_kernel, kMoveGroups, 256, st, m);
}

}  // extern "C"
