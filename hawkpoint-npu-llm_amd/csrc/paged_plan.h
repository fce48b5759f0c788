// How the work of a paged attention is cut into equal runs (plain C++, no HIP:
// also compiled into a test on the CPU).
//
// A task is one tile of an entry's rows (row r: token r / group, query head
// r % group of the kv head) over the blocks of slots that one of them sees.
// Tasks stand in the order entry, kv head, tile.  A task costs task_cost units
// of its own and block_cost for each of its blocks; one that sees nothing has
// an empty block all the same (its rows are still written).  Workgroup w takes
// the blocks that begin in the units [w per, (w + 1) per): whole tasks, and at
// its ends parts of tasks, whose results meet in the workspace.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define HK_PLAN __host__ __device__ inline
#else
#define HK_PLAN inline
#endif

namespace hk {

// A number that is the same in every lane of a wave, in a scalar register.
HK_PLAN int plan_same(int v) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_readfirstlane(v);
#else
  return v;
#endif
}

// x / d for 0 <= x < 2^31 as a product: x * ceil(2^(31 + L) / d) >> (31 + L)
// with 2^L >= d (Granlund and Montgomery, Division by invariant integers using
// multiplication).  A division by a variable is forty instructions.
struct PlanDivisor {
  uint32_t mul;
  int shift;
};
HK_PLAN PlanDivisor plan_divisor(int d) {
  int l = 0;
  while ((1 << l) < d) ++l;
  return {(uint32_t)(((1ull << (31 + l)) + d - 1) / d), 31 + l};
}
HK_PLAN int plan_div(int x, const PlanDivisor& d) { return (int)(((uint64_t)(uint32_t)x * d.mul) >> d.shift); }

struct PlanShape {
  int heads;   // kv heads
  int group;   // query heads per kv head
  PlanDivisor by_group;
  int window;  // 0: none
  int rows;    // of a tile
  int slots;   // of a block
  int block_cost, task_cost;  // units
};

struct PlanEntry {
  int length, count;
};

// The blocks [lo, hi) of a task, and the slots below `seen` that it sees.
struct PlanSpan {
  int lo, hi, seen;
};

HK_PLAN int plan_tiles(const PlanShape& s, const PlanEntry& e) { return (e.count * s.group + s.rows - 1) / s.rows; }

HK_PLAN PlanSpan plan_span(const PlanShape& s, const PlanEntry& e, int tile) {
  const int r0 = tile * s.rows, end = r0 + s.rows < e.count * s.group ? r0 + s.rows : e.count * s.group;
  const int p0 = e.length - e.count + plan_div(r0, s.by_group), p1 = e.length - e.count + plan_div(end - 1, s.by_group);
  const int low = s.window > 0 && p0 >= s.window ? p0 - s.window + 1 : 0;
  if (p1 < low) return {0, 0, 0};
  return {low / s.slots, p1 / s.slots + 1, p1 + 1};
}

HK_PLAN int plan_blocks(const PlanSpan& s) { return s.hi > s.lo ? s.hi - s.lo : 1; }
HK_PLAN int64_t plan_units(const PlanShape& s, const PlanSpan& span) {
  return s.task_cost + (int64_t)s.block_cost * plan_blocks(span);
}

// Units of one kv head of an entry.
HK_PLAN int64_t plan_head_units(const PlanShape& s, const PlanEntry& e) {
  int64_t n = 0;
  const int tiles = plan_tiles(s, e);
  for (int t = 0; t < tiles; ++t) n += plan_units(s, plan_span(s, e, t));
  return n;
}

// a / b of numbers that are not negative, in 32 bits where they fit (on the GPU
// a 64-bit division costs four times as much).
HK_PLAN int64_t plan_div(int64_t a, int64_t b) {
  return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// Units per workgroup; at least a block, so that every workgroup between a
// task's first and last has a block of it.
HK_PLAN int64_t plan_per(const PlanShape& s, int64_t total, int groups, int least) {
  const int64_t per = plan_div(total + groups - 1, groups), most = (int64_t)least * s.block_cost;
  return per > most ? per : most;
}

// A workgroup's run: the units [begin, end).  Consecutive runs are on one XCD
// (workgroups go round the eight), where they share K and V rows in its L2, and
// the XCDs have equally many.
constexpr int kPlanXcds = 8;
struct PlanRun {
  int w;  // its number
  int64_t begin, end, per;
};
// The run of workgroup `block` of `groups`; false: it has none.
HK_PLAN bool plan_cut(const PlanShape& s, int64_t total, int groups, int least, int block, PlanRun& r) {
  r.per = plan_per(s, total, groups, least);
  const int runs = (int)plan_div(total + r.per - 1, r.per), share = (runs + kPlanXcds - 1) / kPlanXcds;
  r.w = block % kPlanXcds * share + block / kPlanXcds;
  r.begin = r.w * r.per;
  r.end = total < r.begin + r.per ? total : r.begin + r.per;
  return block / kPlanXcds < share && r.begin < r.end;
}

// A task's place in the order: `start` units lie before it.
struct PlanPlace {
  int entry, head, tile;
  int64_t start;
};

// The task that unit `rem` of entry `entry` belongs to; the entry starts at
// unit `start`.  (One thread's form: the kernel has the 64 lanes of a wave do
// the same, and this is what the CPU test goes by.)
HK_PLAN PlanPlace plan_find(const PlanShape& s, const PlanEntry& e, int entry, int64_t start, int64_t rem) {
  const int64_t per_head = plan_head_units(s, e);
  PlanPlace p = {entry, (int)plan_div(rem, per_head), 0, 0};
  rem -= p.head * per_head;
  p.start = start + p.head * per_head;
  for (;;) {
    const int64_t u = plan_units(s, plan_span(s, e, p.tile));
    if (rem < u) return p;
    rem -= u;
    p.start += u;
    ++p.tile;
  }
}

// The blocks [first, end) of a task that begin in the units [u0, u1).
struct PlanBlocks {
  int first, end;
};
HK_PLAN int plan_block_at(const PlanShape& s, int64_t start, int blocks, int64_t u) {
  const int64_t past = u - start - s.task_cost;
  if (past <= 0) return 0;
  const int64_t k = plan_div(past + s.block_cost - 1, s.block_cost);
  return k < blocks ? (int)k : blocks;
}
HK_PLAN PlanBlocks plan_mine(const PlanShape& s, int64_t start, int blocks, int64_t u0, int64_t u1) {
  return {plan_block_at(s, start, blocks, u0), plan_block_at(s, start, blocks, u1)};
}

// The workgroups that have blocks of a task, and the place of workgroup w's
// part among the partial results.  Each workgroup has two: for the task that it
// goes on with, and for the one that it begins (whose first block is its own).
struct PlanParts {
  int first, count;
};
HK_PLAN PlanParts plan_parts(const PlanShape& s, int64_t start, int blocks, int64_t per) {
  start += s.task_cost;
  const int first = (int)plan_div(start, per), last = (int)plan_div(start + (int64_t)s.block_cost * (blocks - 1), per);
  return {first, last - first + 1};
}
HK_PLAN int plan_slot(const PlanParts& p, int w) { return 2 * w + (w == p.first ? 1 : 0); }

// On to the next task of a run, if that ends later.  next(place): on to the next
// entry that has rows, if there is one (place.entry, and e).
template <typename Next>
HK_PLAN void plan_next(const PlanShape& s, const PlanEntry& e, PlanPlace& p, int64_t end, Next next) {
  p.start += plan_units(s, plan_span(s, e, p.tile));
  if (p.start >= end) return;
  if (++p.tile < plan_tiles(s, e)) return;
  p.tile = 0;
  if (++p.head < s.heads) return;
  p.head = 0;
  next(p);
}

// A workgroup's part of a task: the blocks `mine` of those of `span`, and the
// parts that it is one of, if it is cut.
struct PlanTask {
  int head, tile;
  PlanSpan span;
  PlanBlocks mine;
  PlanParts parts;
  bool cut;
};

// The task at the place, or the next one of which the run has blocks; take(task)
// is called before the place goes on.  False: there is none.
template <typename Take, typename Next>
HK_PLAN bool plan_take(const PlanShape& s, const PlanRun& r, const PlanEntry& e, PlanPlace& p, Take take, Next next) {
  for (; p.start < r.end; plan_next(s, e, p, r.end, next)) {
    const PlanSpan span = plan_span(s, e, p.tile);
    const int blocks = plan_blocks(span);
    const PlanBlocks mine = plan_mine(s, p.start, blocks, r.begin, r.end);
    if (mine.first >= mine.end) continue;
    const bool cut = mine.end - mine.first < blocks;
    take(PlanTask{p.head, p.tile, span, mine, cut ? plan_parts(s, p.start, blocks, r.per) : PlanParts{0, 0}, cut});
    plan_next(s, e, p, r.end, next);
    return true;
  }
  return false;
}

// A batch of one entry over a long context may be cut another way: every task
// into `splits` parts of as many blocks each (or, of more tasks than
// workgroups, whole tasks dealt out one after the other), so that the
// workgroups of a kv head go through the same slots at the same time and find
// them in their XCD's L2.  Equal runs start all over the context: a context that
// L2 does not hold then comes from memory once for each tile.  (A 2039-token piece
// over 30011 slots: 1113 us, in equal runs 1130 to 1230.  Two of them in a call,
// which have equal runs: 2420 us where one has 1100; two of 1019: 1215 and 583.)
struct PlanEven {
  int splits;  // 0: equal runs
  int tasks;
};
// Taken where the longest workgroup has at most a quarter more than the average
// (an entry without a past has tiles of one block and of all: half the
// workgroups would wait).  `total`: units of all tasks.
HK_PLAN PlanEven plan_even(const PlanShape& s, const PlanEntry& e, int64_t total, int groups) {
  const int tiles = plan_tiles(s, e), tasks = s.heads * tiles;
  const int splits = tasks <= groups ? groups / tasks : 1, rounds = (tasks + groups - 1) / groups;
  const int blocks = plan_blocks(plan_span(s, e, tiles - 1));
  const int64_t longest = rounds * (s.task_cost + (int64_t)s.block_cost * ((blocks + splits - 1) / splits));
  return {4 * longest * groups <= 5 * total ? splits : 0, tasks};
}

// Part `part` of `splits` of a task's blocks, and the parts that have some.
HK_PLAN int plan_even_parts(int blocks, int splits) { return blocks < splits ? blocks : splits; }
HK_PLAN PlanBlocks plan_even_mine(int blocks, int splits, int part) {
  const int parts = plan_even_parts(blocks, splits);
  if (part >= parts) return {0, 0};
  return {(int)((int64_t)blocks * part / parts), (int)((int64_t)blocks * (part + 1) / parts)};
}

// The number that workgroup `block` has in the even cut, neighbours on one XCD.
HK_PLAN int plan_even_number(int block, int groups) { return block % kPlanXcds * (groups / kPlanXcds) + block / kPlanXcds; }

// The part of task `next` that workgroup number w has, and its next task; false:
// there is none.
HK_PLAN bool plan_even_take(const PlanShape& s, const PlanEntry& e, const PlanEven& even, int w, int groups, int& next,
                            PlanTask& t) {
  if (next >= even.tasks) return false;
  const int tiles = plan_tiles(s, e), task = next;
  t.head = plan_same(task / tiles);
  t.tile = task - t.head * tiles;
  t.span = plan_span(s, e, t.tile);
  const int blocks = plan_blocks(t.span);
  t.parts = {task * even.splits, plan_even_parts(blocks, even.splits)};
  // (whole tasks: the workgroup's number plays no part)
  t.mine = even.splits == 1 ? PlanBlocks{0, blocks} : plan_even_mine(blocks, even.splits, w - task * even.splits);
  t.cut = t.mine.end - t.mine.first < blocks;
  next += even.splits == 1 ? groups : even.tasks;
  return t.mine.first < t.mine.end;
}

}  // namespace hk
