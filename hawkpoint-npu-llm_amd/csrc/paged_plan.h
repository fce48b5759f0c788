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

// A task's place in the order: `start` units lie before it.
struct PlanPlace {
  int entry, head, tile;
  int64_t start;
};

// The task that unit `rem` of entry `entry` belongs to; the entry starts at
// unit `start`.
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

// A batch of one entry over a long context may be cut another way: every task
// into `splits` parts of as many blocks each (or, of more tasks than
// workgroups, whole tasks dealt out one after the other), so that the
// workgroups of a kv head go through the same slots at the same time and find
// them in their XCD's L2.  Equal runs start all over the context: a context that
// L2 does not hold then comes from memory once for each tile.
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

}  // namespace hk
