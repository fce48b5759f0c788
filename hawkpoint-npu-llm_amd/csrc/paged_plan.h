// How the work of a paged attention is cut into equal runs (plain C++, no HIP:
// also compiled into a test on the CPU).
//
// A task is one tile of an entry's rows (row r: token r / group, query head
// r % group of the kv head) over the blocks of slots that one of them sees.
// Tasks stand in the order entry, kv head, tile; a block is a unit of work, a
// task that sees nothing one unit too (its rows are still written).  Workgroup
// w takes the units [w per, (w + 1) per): whole tasks, and at its ends parts of
// tasks, whose results meet in the workspace.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define HK_PLAN __host__ __device__ inline
#else
#define HK_PLAN inline
#endif

namespace hk {

struct PlanShape {
  int heads;   // kv heads
  int group;   // query heads per kv head
  int window;  // 0: none
  int rows;    // of a tile
  int slots;   // of a block
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
  const int p0 = e.length - e.count + r0 / s.group, p1 = e.length - e.count + (end - 1) / s.group;
  const int low = s.window > 0 && p0 >= s.window ? p0 - s.window + 1 : 0;
  if (p1 < low) return {0, 0, 0};
  return {low / s.slots, p1 / s.slots + 1, p1 + 1};
}

HK_PLAN int plan_units(const PlanSpan& s) { return s.hi > s.lo ? s.hi - s.lo : 1; }

// Units of one kv head of an entry.
HK_PLAN int64_t plan_head_units(const PlanShape& s, const PlanEntry& e) {
  int64_t n = 0;
  const int tiles = plan_tiles(s, e);
  for (int t = 0; t < tiles; ++t) n += plan_units(plan_span(s, e, t));
  return n;
}

// a / b of numbers that are not negative, in 32 bits where they fit (on the GPU
// a 64-bit division costs four times as much).
HK_PLAN int64_t plan_div(int64_t a, int64_t b) {
  return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

HK_PLAN int64_t plan_per(int64_t total, int groups, int least) {
  const int64_t per = plan_div(total + groups - 1, groups);
  return per > least ? per : least;
}

// A place in the order of tasks: `at` units of the task lie before it, `start`
// units before the task.
struct PlanPlace {
  int entry, head, tile;
  int at;
  int64_t start;
};

// The place `rem` units into entry `entry`, which starts at unit `start`.
HK_PLAN PlanPlace plan_find(const PlanShape& s, const PlanEntry& e, int entry, int64_t start, int64_t rem) {
  const int64_t per_head = plan_head_units(s, e);
  PlanPlace p = {entry, (int)plan_div(rem, per_head), 0, 0, 0};
  rem -= p.head * per_head;
  start += p.head * per_head;
  for (;;) {
    const int u = plan_units(plan_span(s, e, p.tile));
    if (rem < u) break;
    rem -= u;
    start += u;
    ++p.tile;
  }
  p.at = (int)rem;
  p.start = start;
  return p;
}

// Parts of a task of `units` units from `start`: the workgroups that have
// some, and the place of workgroup w's part among the partial results (two
// per workgroup: the task it goes on with, and the task it begins).
struct PlanParts {
  int first, count;
};
HK_PLAN PlanParts plan_parts(int64_t start, int units, int64_t per) {
  const int first = (int)plan_div(start, per), last = (int)plan_div(start + units - 1, per);
  return {first, last - first + 1};
}
HK_PLAN int plan_slot(int64_t start, int w, int64_t per) { return 2 * w + (start >= w * per ? 1 : 0); }

}  // namespace hk
