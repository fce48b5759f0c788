"""The paged cache without a GPU: the exports and binding of include/hk_paged.h, what the calls refuse before any
device work, and the float64 oracle against other formulations."""

import ctypes
import os
import re
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from oracle import paged as oracle

ROOT = Path(__file__).resolve().parents[1]


def test_exports_and_binding():
    from runtime import hip, paged

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "hk_paged.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(hk_paged_[a-z0-9_]+)\s*\(", text))
    assert names == set(paged.EXPORTED) == {"hk_paged_append", "hk_paged_attention", "hk_paged_fork",
                                            "hk_paged_compact"}
    lib = ctypes.CDLL(str(hip.LIB_PATH))
    assert all(hasattr(lib, n) for n in names)
    assert int(re.search(r"HK_PAGED_WORKSPACE (\d+)", text).group(1)) == paged.WORKSPACE
    fields = re.search(r"typedef struct hk_paged_cache \{(.*?)\}", text, flags=re.S).group(1)
    assert re.findall(r"(\w+);", fields) == [n for n, _ in paged.PagedCache._fields_]


# Host memory stands in for device pointers: a refused call never looks at it.
HERE = (ctypes.c_char * 4096)()
AT = -(-ctypes.addressof(HERE) // 256) * 256


def _cache(**changes):
    from runtime import paged

    c = dict(k=AT, v=AT, k_scale=None, v_scale=None, table=AT, length=AT, refs=AT, layer_stride=1 << 20,
             page_stride=2 * 16 * 64, layers=2, kv_heads=2, head_dim=64, page_size=16, pages=8, seqs=4, table_width=4,
             dtype=paged.BF16)
    c.update(changes)
    return paged.PagedCache(**c)


APPEND = dict(layer=0, qkv=AT, qkv_stride=512, cos=AT, sin=AT, positions=64, seqs=AT, first=AT, n=2, tokens=3,
              q_heads=4, q_out=AT + 1024, q_out_stride=256, stream=None)
ATTENTION = dict(layer=0, q=AT, q_stride=256, seqs=AT, first=AT, n=2, tokens=3, max_new=2, q_heads=4, scale=0.125,
                 window=0, out=AT, out_stride=256, lse=None, workspace=AT, stream=None)
FORK = dict(child=None, parent=None, keep=None, grow=None, n=2, status=AT, workspace=AT, stream=None)
COMPACT = dict(table_out=AT, refs_out=AT, live_out=AT, workspace=AT, stream=None)
CALLS = {"hk_paged_append": APPEND, "hk_paged_attention": ATTENTION, "hk_paged_fork": FORK, "hk_paged_compact": COMPACT}


def _refused(name, cache, rc, **changes):
    from runtime import hip, paged

    args = dict(CALLS[name], **changes)
    got = getattr(paged.lib(), name)(None if cache is None else ctypes.byref(cache), *args.values())
    assert got == rc, (got, hip.last_error())
    assert hip.last_error().startswith(name)


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refuses_bad_caches(name):
    from runtime import hip, paged

    bad, unsupported = hip.HK_ERR_INVALID, hip.HK_ERR_UNSUPPORTED
    _refused(name, None, bad)
    for field in ("k", "v", "table", "length", "refs"):
        _refused(name, _cache(**{field: None}), bad)
    for changes, rc in ((dict(head_dim=96), unsupported), (dict(page_size=8), unsupported),
                        (dict(page_size=48), unsupported), (dict(page_size=512), unsupported), (dict(dtype=2), bad),
                        (dict(layers=0), bad), (dict(kv_heads=0), bad), (dict(pages=0), bad), (dict(seqs=-1), bad),
                        (dict(table_width=0), bad), (dict(table_width=1 << 27), bad),
                        (dict(page_stride=2 * 16 * 64 - 8), bad), (dict(page_stride=2 * 16 * 64 + 4), bad),
                        (dict(layer_stride=2 * 16 * 64 - 8), bad), (dict(layer_stride=2 * 16 * 64 + 1), bad),
                        (dict(k=AT + 8), bad), (dict(v=AT + 2), bad), (dict(dtype=paged.E4M3), bad),
                        (dict(dtype=paged.E4M3, k_scale=AT), bad),
                        (dict(dtype=paged.E4M3, k_scale=AT, v_scale=AT, page_stride=2 * 16 * 64 + 8), bad)):
        _refused(name, _cache(**changes), rc)


@pytest.mark.parametrize("name", ["hk_paged_append", "hk_paged_attention"])
def test_refuses_bad_batches(name):
    from runtime import hip

    for changes in (dict(layer=-1), dict(layer=2), dict(first=None), dict(n=-1), dict(tokens=-1), dict(n=4097),
                    dict(q_heads=3), dict(q_heads=0), dict(q_heads=8192)):
        _refused(name, _cache(), hip.HK_ERR_INVALID, **changes)


def test_refuses_bad_arguments():
    from runtime import hip, paged

    bad = hip.HK_ERR_INVALID
    for changes in (dict(qkv=None), dict(qkv=AT + 2), dict(qkv_stride=511), dict(qkv_stride=504), dict(q_out=AT + 8),
                    dict(q_out_stride=248), dict(cos=None), dict(sin=None), dict(sin=AT + 4), dict(positions=63),
                    dict(q_out_stride=256, q_out=APPEND["qkv"], qkv_stride=520)):
        _refused("hk_paged_append", _cache(), bad, **changes)
    for changes in (dict(q=None), dict(out=None), dict(q=AT + 8), dict(out=AT + 4), dict(q_stride=248),
                    dict(out_stride=260), dict(workspace=None), dict(workspace=AT + 16), dict(max_new=0),
                    dict(out=AT, out_stride=264), dict(window=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                    dict(scale=float("inf"))):
        _refused("hk_paged_attention", _cache(), bad, **changes)
    _refused("hk_paged_append", _cache(), hip.HK_ERR_UNSUPPORTED, tokens=1 << 24)
    _refused("hk_paged_attention", _cache(), hip.HK_ERR_UNSUPPORTED, tokens=(1 << 28) + 1)
    for changes in (dict(status=None), dict(workspace=None), dict(workspace=AT + 8), dict(n=0), dict(n=5)):
        _refused("hk_paged_fork", _cache(), bad, **changes)
    _refused("hk_paged_fork", _cache(seqs=30000, table_width=1000), hip.HK_ERR_UNSUPPORTED, n=30000)
    for changes in (dict(table_out=None), dict(refs_out=None), dict(live_out=None), dict(workspace=None)):
        _refused("hk_paged_compact", _cache(), bad, **changes)
    _refused("hk_paged_compact", _cache(pages=1 << 24), hip.HK_ERR_UNSUPPORTED)
    # nothing to do is no error
    for name in ("hk_paged_append", "hk_paged_attention"):
        for changes in (dict(n=0), dict(tokens=0)):
            args = dict(CALLS[name], **changes)
            assert getattr(paged.lib(), name)(ctypes.byref(_cache()), *args.values()) == hip.HK_OK


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refuses_misaligned_arrays(name):
    """Vector and scalar loads would read different numbers from them."""
    from runtime import hip, paged

    for field in ("table", "length", "refs", "status"):
        for off in (1, 2, 3):
            _refused(name, _cache(**{field: AT + off}), hip.HK_ERR_INVALID)
    for scales in (dict(k_scale=AT + 2, v_scale=AT), dict(k_scale=AT, v_scale=AT + 1)):
        _refused(name, _cache(dtype=paged.E4M3, **scales), hip.HK_ERR_INVALID)
    for arg in ("seqs", "first", "lse", "child", "parent", "keep", "grow", "status", "table_out", "refs_out", "live_out"):
        if arg in CALLS[name]:
            _refused(name, _cache(), hip.HK_ERR_INVALID, **{arg: AT + 2})


CHILD = """
import ctypes, sys
fake = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # before libhk.so: its calls go here
from runtime import hip, paged
hip.init(0)
lib = paged.lib()
b = hip.DeviceBuffer(1 << 16)
at = -(-b.ptr // 256) * 256
stream = ctypes.c_void_p()
hip.check(lib.hk_stream_create(ctypes.byref(stream)), "stream")
c = ctypes.byref(paged.PagedCache(k=at, v=at, table=at, length=at, refs=at, layer_stride=4096, page_stride=2048, layers=2,
                                  kv_heads=2, head_dim=64, page_size=16, pages=8, seqs=4, table_width=4, dtype=paged.BF16))
calls = {
    "append": lambda: lib.hk_paged_append(c, 1, at, 512, at, at, 64, None, at, 2, 3, 4, at + 1024, 256, stream),
    "token": lambda: lib.hk_paged_attention(c, 1, at, 256, None, at, 2, 3, 1, 4, 0.125, 0, at, 256, None, at, stream),
    "mixed": lambda: lib.hk_paged_attention(c, 1, at, 256, None, at, 2, 300, 99, 4, 0.125, 0, at, 256, None, at, stream),
    "pieces": lambda: lib.hk_paged_attention(c, 1, at, 4096, None, at, 2, 300, 99, 64, 0.125, 0, at, 4096, None, at, stream),
    "fork": lambda: lib.hk_paged_fork(c, None, None, None, None, 2, at, at, stream),
    "compact": lambda: lib.hk_paged_compact(c, at, at, at, at, stream),
}
before = fake.fake_device_bytes()
for name, call in calls.items():
    assert call() == 0, hip.last_error()
    for launch in range(2 if name in ("pieces", "fork", "compact") else 1):
        fake.fake_fail_launch(launch)
        assert call() == hip.HK_ERR_HIP and "paged" in hip.last_error(), (name, launch, hip.last_error())
        fake.fake_fail_launch(-1)
        assert call() == 0, (name, hip.last_error())
assert fake.fake_device_bytes() == before, "a call allocated device memory"
"""


def test_calls_allocate_nothing_and_report_failed_launches(tmp_path):
    """Over the runtime of _fake_hip.cpp, where no kernel runs: the calls make no allocation, and a launch that fails is
    that call's error and no later one's."""
    lib = tmp_path / "libfakehip.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    str(ROOT / "tests" / "_fake_hip.cpp"), "-o", str(lib)], check=True)
    path = os.pathsep.join([str(ROOT), str(ROOT / "hawkpoint-npu-llm_amd")])
    done = subprocess.run([sys.executable, "-c", CHILD, str(lib)], capture_output=True, text=True, timeout=120,
                          env={**os.environ, "PYTHONPATH": path})
    assert done.returncode == 0, done.stdout + done.stderr


# ---- the oracle ----


def test_oracle_e4m3_rounds_to_nearest_even():
    torch = pytest.importorskip("torch")
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(oracle.from_e4m3(codes), want)
    rng = np.random.default_rng(0)
    steps = oracle.from_e4m3(np.arange(127))
    x = np.concatenate((rng.normal(0, 50, 4000), rng.normal(0, 0.01, 4000), (steps[1:] + steps[:-1]) / 2, steps, -steps,
                        [448.0, 463.9, 0.0, -0.0]))
    x = x.astype(np.float32)
    got = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(oracle.e4m3(x), got)
    assert oracle.e4m3(np.nan) == 0x7F and oracle.e4m3(np.inf) == 0x7E and oracle.e4m3(-1e9) == 0xFE


def _random_cache(rng, layers=1, pages=12, heads=2, page=16, dim=64, seqs=4, width=6):
    return {"k": rng.normal(size=(layers, pages, heads, page, dim)), "v": rng.normal(size=(layers, pages, heads, page, dim)),
            "table": np.full((seqs, width), -1, np.int32), "length": np.zeros(seqs, np.int32),
            "refs": np.zeros(pages, np.int32)}


def test_oracle_attention_is_softmax_over_the_visible_slots():
    rng = np.random.default_rng(1)
    c = _random_cache(rng)
    c["table"][0, :3], c["length"][0] = (7, 2, 9), 41
    q = rng.normal(size=(5, 4, 64))
    k = np.concatenate([c["k"][0, p] for p in (7, 2, 9)], 1)[:, :41]
    v = np.concatenate([c["v"][0, p] for p in (7, 2, 9)], 1)[:, :41]
    for window in (0, 1, 20):
        out, lse, spread = oracle.attention(c, 0, q, [0], [0, 5], 0.3, window)
        for t in range(5):
            lo = max(0, 36 + t - window + 1) if window else 0
            for h in range(4):
                s = 0.3 * k[h // 2, lo:37 + t] @ q[t, h]
                p = np.exp(s) / np.exp(s).sum()
                np.testing.assert_allclose(out[t, h], p @ v[h // 2, lo:37 + t], rtol=1e-12, atol=1e-12)
                np.testing.assert_allclose(lse[t, h], np.log(np.exp(s).sum()), rtol=1e-12)
    # a planted mistake is caught: one slot more
    assert np.abs(oracle.attention(c, 0, q, [0], [0, 4], 0.3)[0][:4] - out[:4]).max() > 1e-3
    # rows before the first token, rows of no entry, an absent page
    c["length"][0] = 2
    out, lse, _ = oracle.attention(c, 0, q, [0, 9], [0, 4, 5], 1.0)
    assert np.all(out[:2] == 0) and np.all(lse[:2] == -np.inf) and np.all(lse[4] == -np.inf)
    np.testing.assert_array_equal(out[2, 0], v[0, 0])


def _held(c):
    """refs as the tables say."""
    n = np.zeros(len(c["refs"]), np.int64)
    for s, length in enumerate(c["length"]):
        for p in c["table"][s, :-(-length // c["k"].shape[3])]:
            n[p] += 1
    return n


def _tokens(c, s):
    """What a sequence says: its key rows in order."""
    page = c["k"].shape[3]
    return np.concatenate([c["k"][:, p] for p in c["table"][s, :-(-c["length"][s] // page)]] or [c["k"][:, 0][:, :, :0]],
                          2)[:, :, :c["length"][s]]


def test_oracle_fork_keeps_contents_and_counts():
    rng = np.random.default_rng(2)
    c = _random_cache(rng, layers=2, pages=16)
    free = lambda: int((c["refs"] == 0).sum())  # noqa: E731
    assert oracle.fork(c, [0, 1], [0, 1], [0, 0], [37, 16]) == (0, 0)
    assert c["length"].tolist() == [37, 16, 0, 0] and free() == 16 - 4
    told = _tokens(c, 0)
    assert oracle.fork(c, [2, 3, 0], [0, 0, 0], [37, 20, 37], [0, 1, 1]) == (0, 0)
    # two full pages shared; 2 and 0 differ in the last page, 3 copied 4 slots of the second
    assert c["refs"].tolist() == _held(c).tolist() and sorted(c["refs"])[-1] == 3
    for s, n in ((0, 37), (2, 37), (3, 20)):
        np.testing.assert_array_equal(_tokens(c, s)[:, :, :n], told[:, :, :n])
    # beams reordered: everyone's parent is another child
    before = [_tokens(c, s) for s in range(4)]
    keep = c["length"].tolist()
    assert oracle.fork(c, [0, 1, 2, 3], [1, 2, 3, 0], keep[1:] + keep[:1], [0] * 4) == (0, 0)
    for s in range(4):
        np.testing.assert_array_equal(_tokens(c, s), before[(s + 1) % 4])
    assert c["refs"].tolist() == _held(c).tolist()
    # what is not valid, and too little room, changes nothing
    state = {x: c[x].copy() for x in c}
    n = [int(x) for x in c["length"]]
    for args, status in ((([0, 0], [0, 0], [0, 0], [0, 0]), (1, 1)), (([4], [0], [0], [0]), (1, 0)),
                         (([0], [0], [n[0] + 1], [0]), (1, 0)), (([1, 0], [1, 9], [n[1], 1], [0, 0]), (1, 1)),
                         (([0], [0], [n[0]], [96]), (1, 0)), (([0], [0], [-1], [0]), (1, 0))):
        assert oracle.fork(c, *args) == status
    code, missing = oracle.fork(c, [0, 1, 2, 3], [0, 1, 2, 3], n, [96 - x for x in n])
    assert code == 2 and missing > 0
    for x in state:
        np.testing.assert_array_equal(c[x], state[x])
    # compaction and freeing
    told = [_tokens(c, s) for s in range(4)]
    live = oracle.compact(c)
    assert live == (c["refs"] > 0).sum() and np.all(c["refs"][:live] > 0)
    for s in range(4):
        np.testing.assert_array_equal(_tokens(c, s), told[s])
    assert oracle.fork(c, [0, 1, 2, 3], [9] * 4, [0] * 4, [0] * 4) == (0, 0) and free() == 16


# ---- the cut of the attention's work ----

PLAN = """
#include "paged_plan.h"
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>
using namespace hk;
#define CHECK(x) if (!(x)) { std::printf("%s, seed %d\\n", #x, seed); return 1; }
int main() {
  for (int d = 1, seed = 0; d <= 4096; ++d)
    for (int64_t q = 0; q <= INT32_MAX / d; q = q < 20 || q * d > INT32_MAX - 20 * d ? q + 1 : q + INT32_MAX / d / 7)
      for (int64_t x : {q * d, q * d + d - 1})
        if (x <= INT32_MAX) CHECK(plan_div((int)x, plan_divisor(d)) == x / d);
  for (int seed = 0; seed < 400; ++seed) {
    std::mt19937 rng(seed);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    const int rows[] = {16, 32, 64, 256}, slots[] = {64, 128};
    const int group = pick(1, 9);
    PlanShape s{pick(1, 4), group, plan_divisor(group), pick(0, 2) ? 0 : pick(1, 300), rows[pick(0, 3)], slots[pick(0, 1)], pick(1, 3),
                pick(0, 5)};
    std::vector<PlanEntry> e(pick(1, 12));
    for (auto& x : e) x = {pick(0, 3) ? pick(0, 2000) : 0, pick(0, 3) ? pick(0, 3) : pick(0, 700)};
    int64_t total = 0;
    std::vector<int64_t> start;
    for (auto& x : e) start.push_back(total), total += s.heads * plan_head_units(s, x);
    const int groups = pick(1, 40);
    const int64_t per = plan_per(s, total, groups, pick(1, 4));
    CHECK(groups * per >= total);
    std::map<std::tuple<int, int, int>, std::vector<int>> got;  // task: blocks
    std::map<std::tuple<int, int, int>, int> arrived, asked, ticket;
    std::set<int> partials;
    for (int w = 0; w < groups; ++w) {
      const int64_t begin = w * per, end = std::min(total, begin + per);
      if (begin >= end) continue;
      size_t i = 0;
      while (i + 1 < e.size() && start[i + 1] <= begin) ++i;
      PlanPlace p = plan_find(s, e[i], (int)i, start[i], begin - start[i]);
      CHECK(p.start <= begin);
      while (p.entry < (int)e.size() && p.start < end) {
        const PlanSpan span = plan_span(s, e[p.entry], p.tile);
        const int blocks = plan_blocks(span);
        const PlanBlocks mine = plan_mine(s, p.start, blocks, begin, end);
        const PlanParts parts = plan_parts(s, p.start, blocks, per);
        const auto task = std::make_tuple(p.entry, p.head, p.tile);
        CHECK((mine.first < mine.end) == (w >= parts.first && w < parts.first + parts.count));
        for (int k = mine.first; k < mine.end; ++k) got[task].push_back(k);
        if (mine.first < mine.end && mine.end - mine.first < blocks) {
          const int slot = plan_slot(parts, w);
          CHECK(parts.count > 1 && partials.insert(slot).second && slot < 2 * groups);
          CHECK(!ticket.count(task) || ticket[task] == parts.first);
          ticket[task] = parts.first, asked[task] = parts.count, ++arrived[task];
        }
        p.start += plan_units(s, span);
        if (++p.tile >= plan_tiles(s, e[p.entry])) {
          p.tile = 0;
          if (++p.head >= s.heads) {
            p.head = 0, ++p.entry;
            while (p.entry < (int)e.size() && e[p.entry].count == 0) ++p.entry;
          }
        }
      }
    }
    std::set<int> tickets;
    for (auto& t : ticket) CHECK(tickets.insert(t.second).second && asked[t.first] == arrived[t.first]);
    // every task once, its blocks in order; every slot that a row sees inside a block of its tile
    size_t tasks = 0;
    for (size_t i = 0; i < e.size(); ++i)
      for (int t = 0; t < plan_tiles(s, e[i]); ++t) {
        const PlanSpan span = plan_span(s, e[i], t);
        tasks += s.heads;
        for (int h = 0; h < s.heads; ++h) {
          const auto& blocks = got[std::make_tuple((int)i, h, t)];
          CHECK((int)blocks.size() == plan_blocks(span));
          for (size_t k = 0; k < blocks.size(); ++k) CHECK(blocks[k] == (int)k);
        }
        for (int r = t * s.rows; r < std::min((t + 1) * s.rows, e[i].count * s.group); ++r) {
          const int p = e[i].length - e[i].count + r / s.group, low = s.window ? std::max(0, p - s.window + 1) : 0;
          if (p < 0) continue;
          CHECK(span.lo * s.slots <= low && p < span.hi * s.slots && p < span.seen && span.seen <= e[i].length);
        }
      }
    CHECK(tasks == got.size());
    // the even cut of each entry by itself
    for (auto& x : e) {
      if (!x.count) continue;
      const PlanEven even = plan_even(s, x, s.heads * plan_head_units(s, x), groups);
      if (!even.splits) continue;
      const int tiles = plan_tiles(s, x);
      CHECK(even.tasks == s.heads * tiles && (even.splits == 1 || even.splits * even.tasks <= groups));
      for (int task = 0; task < even.tasks; ++task) {
        const int blocks = plan_blocks(plan_span(s, x, task % tiles)), parts = plan_even_parts(blocks, even.splits);
        int next = 0;
        for (int part = 0; part < even.splits; ++part) {
          const PlanBlocks mine = plan_even_mine(blocks, even.splits, part);
          CHECK((mine.first < mine.end) == (part < parts));
          if (part < parts) CHECK(mine.first == next);
          if (part < parts) next = mine.end;
        }
        CHECK(next == blocks && parts >= 1);
      }
    }
  }
}
"""


def test_every_block_of_every_task_has_one_workgroup(tmp_path):
    """csrc/paged_plan.h on random batches: the runs cover every task's blocks once and in order, no two parts share a
    place in the workspace, the tasks' tickets are their own and count the parts that arrive."""
    (tmp_path / "plan.cpp").write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'hawkpoint-npu-llm_amd' / 'csrc'}",
                    str(tmp_path / "plan.cpp"), "-o", str(tmp_path / "plan")], check=True)
    done = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


# ---- errors that are not the call's own ----

CHILD_STALE = CHILD[:CHILD.index("before =")] + """
count = {"pieces": 2, "fork": 2, "compact": 2}
p = ctypes.c_void_p()
for name, call in calls.items():
    # the caller's own HIP use has failed, and it has dealt with that: HIP keeps the error for the next who asks
    fake.fake_fail_malloc_after(0)
    assert fake.hipMalloc(ctypes.byref(p), ctypes.c_size_t(64)) != 0
    fake.fake_fail_launch(count.get(name, 1))
    assert call() == 0, (name, hip.last_error())
    # all its launches were made: the next launch of all is the one to fail
    assert calls["append"]() == hip.HK_ERR_HIP, name
    fake.fake_fail_launch(-1)
"""


def test_an_earlier_hip_error_of_the_callers_stops_no_call(tmp_path):
    """A fork that took it for its own would leave tables that name pages nobody has copied."""
    lib = tmp_path / "libfakehip.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    str(ROOT / "tests" / "_fake_hip.cpp"), "-o", str(lib)], check=True)
    path = os.pathsep.join([str(ROOT), str(ROOT / "hawkpoint-npu-llm_amd")])
    done = subprocess.run([sys.executable, "-c", CHILD_STALE, str(lib)], capture_output=True, text=True, timeout=120,
                          env={**os.environ, "PYTHONPATH": path})
    assert done.returncode == 0, done.stdout + done.stderr


CHILD_STREAMS = """
import ctypes, sys
fake = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # before libhk.so: its calls go here
import numpy as np
from runtime import hip, paged
kv = paged.PagedKV(layers=1, kv_heads=2, head_dim=64, page_size=16, pages=8, seqs=4, table_width=4)
lib = paged.lib()
at = hip.DeviceBuffer(1 << 16).ptr
calls = {
    "append": lambda s: kv.append(0, at, [0, 1], [0, 1, 3], 4, q_out=at + 8192, stream=s),
    "attention": lambda s: kv.attention(0, at, [0, 1], [0, 1, 3], 4, at, stream=s),
    "release": lambda s: kv.release([2], s),
    "extend": lambda s: kv.extend([2], [0], s),
    "compact": lambda s: kv.compact(s),
    "lengths": lambda s: kv.lengths(s),
}
for first in calls.values():
    for second in calls.values():
        handle = ctypes.c_void_p()
        hip.check(lib.hk_stream_create(ctypes.byref(handle)), "create")
        first(handle.value)
        hip.check(lib.hk_stream_sync(handle.value), "sync")
        hip.check(lib.hk_stream_destroy(handle.value), "destroy")
        second(None)
        assert fake.fake_dead_streams() == 0
# a call waits for the one before, whose stream it may not know any more
handle = ctypes.c_void_p()
hip.check(lib.hk_stream_create(ctypes.byref(handle)), "create")
before = fake.fake_unwaited()
calls["append"](handle.value)
assert fake.fake_unwaited() == before + 1
calls["attention"](None)
assert fake.fake_unwaited() == before + 1  # the append's work is done, the attention's is not
kv.close()
"""

# _fake_hip.cpp, whose streams go on living when they are destroyed, with handles that end, launches that take until
# something waits for them, and events.
FAKE_STREAMS = """
#define hipStreamCreateWithFlags base_create
#define hipStreamDestroy base_destroy
#define hipStreamSynchronize base_sync
#define hipLaunchKernel base_launch
#define hipMalloc base_malloc
#include "_fake_hip.cpp"
#undef hipStreamCreateWithFlags
#undef hipStreamDestroy
#undef hipStreamSynchronize
#undef hipLaunchKernel
#undef hipMalloc
#include <set>
namespace {
std::set<hipStream_t> live = {nullptr};
std::map<hipStream_t, long> made, waited;  // launches of a stream, and those of them that are done
struct Mark { hipStream_t s; long upto; };
long dead = 0;
bool known(hipStream_t s) { return live.count(s) ? true : (++dead, false); }
}
extern "C" {
long fake_dead_streams() { return dead; }
long fake_unwaited() { long n = 0; for (auto& m : made) n += m.second - waited[m.first]; return n; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned f) { const hipError_t e = base_create(s, f); live.insert(*s); return e; }
hipError_t hipStreamDestroy(hipStream_t s) { if (!known(s)) return note(hipErrorInvalidHandle); live.erase(s); return base_destroy(s); }
hipError_t hipStreamSynchronize(hipStream_t s) {
  if (!known(s)) return note(hipErrorInvalidHandle);
  waited[s] = made[s];
  return base_sync(s);
}
hipError_t hipLaunchKernel(const void* f, dim3 g, dim3 b, void** a, size_t n, hipStream_t s) {
  if (!known(s)) return note(hipErrorInvalidHandle);
  ++made[s];
  return base_launch(f, g, b, a, n, s);
}
hipError_t hipMalloc(void** p, size_t n) {  // aligned as device memory is
  *p = std::aligned_alloc(256, n / 256 * 256 + 256);
  std::memset(*p, 0, n);
  device[static_cast<char*>(*p)] = n;
  return hipSuccess;
}
hipError_t hipEventCreate(hipEvent_t* e) { *e = reinterpret_cast<hipEvent_t>(new Mark{nullptr, -1}); return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t e) { delete reinterpret_cast<Mark*>(e); return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) {
  if (!known(s)) return note(hipErrorInvalidHandle);
  *reinterpret_cast<Mark*>(e) = {s, made[s]};
  return hipSuccess;
}
hipError_t hipEventSynchronize(hipEvent_t e) {
  const Mark& m = *reinterpret_cast<Mark*>(e);
  if (waited[m.s] < m.upto) waited[m.s] = m.upto;
  finish_stream(m.s);
  return hipSuccess;
}
hipError_t hipEventElapsedTime(float* ms, hipEvent_t a, hipEvent_t b) {
  *ms = 0;
  return reinterpret_cast<Mark*>(a)->upto < 0 || reinterpret_cast<Mark*>(b)->upto < 0 ? note(hipErrorInvalidHandle) : hipSuccess;
}
}
"""


def test_cache_outlives_the_streams_of_its_calls(tmp_path):
    """PagedKV waits for the call before, whose stream the caller may have destroyed by then."""
    (tmp_path / "fake.cpp").write_text(FAKE_STREAMS)
    lib = tmp_path / "libfakehip.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-I{ROOT / 'tests'}", str(tmp_path / "fake.cpp"), "-o", str(lib)], check=True)
    path = os.pathsep.join([str(ROOT), str(ROOT / "hawkpoint-npu-llm_amd")])
    done = subprocess.run([sys.executable, "-c", CHILD_STREAMS, str(lib)], capture_output=True, text=True, timeout=120,
                          env={**os.environ, "PYTHONPATH": path})
    assert done.returncode == 0, done.stdout + done.stderr


# ---- the walk of the attention's workgroups ----

WALK = """
#include "paged_plan.h"
#include <algorithm>
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>
using namespace hk;
#define CHECK(x) if (!(x)) { std::printf("%s, seed %d\\n", #x, seed); return 1; }
using Key = std::tuple<int, int, int>;  // entry, head, tile
int main() {
  int evens = 0, rounds = 0;
  for (int seed = 0; seed < 1500; ++seed) {
    std::mt19937 rng(seed);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    const int rows[] = {16, 32, 128}, slots[] = {64, 128}, group = pick(1, 9);
    PlanShape s{pick(1, 6), group, plan_divisor(group), pick(0, 2) ? 0 : pick(1, 300), rows[pick(0, 2)], slots[pick(0, 1)], pick(1, 3),
                pick(0, 5)};
    std::vector<PlanEntry> e(seed % 3 ? pick(1, 12) : 1);
    for (auto& x : e) x = {pick(0, 3) ? pick(0, 4000) : 0, pick(0, 3) ? pick(0, 3) : pick(0, 700)};
    if (e.size() == 1) e[0].count = pick(1, 300);
    // the entries of one of two forms
    const int least_rows = pick(0, 1) ? 1 : 17, most_rows = least_rows == 1 && pick(0, 1) ? 16 : INT32_MAX;
    auto takes = [&](const PlanEntry& x) { return x.count > 0 && x.count * group >= least_rows && x.count * group <= most_rows; };
    const int groups = 8 * pick(1, 40), n = (int)e.size(), least = pick(0, 1) ? 1 : 4;
    int64_t total = 0;
    std::vector<int64_t> start;
    for (auto& x : e) start.push_back(total), total += takes(x) ? s.heads * plan_head_units(s, x) : 0;
    std::map<Key, std::vector<std::pair<int, PlanBlocks>>> got;  // who, blocks
    std::map<Key, int> count, ticket;
    std::set<int> places, tickets, numbers;
    auto arrived = [&](const Key& key, int who, const PlanTask& t, int blocks) {
      got[key].push_back({who, t.mine});
      if (t.mine.first >= t.mine.end || t.cut != (t.mine.end - t.mine.first < blocks)) return false;
      if (!t.cut) return true;
      const int place = plan_slot(t.parts, who);
      if (place < 0 || place >= 2 * groups || !places.insert(place).second || t.parts.first < 0 || t.parts.first >= groups) return false;
      if (!count.count(key)) {
        count[key] = t.parts.count, ticket[key] = t.parts.first;
        return tickets.insert(t.parts.first).second;
      }
      return count[key] == t.parts.count && ticket[key] == t.parts.first;
    };
    PlanEven even = {0, 0};
    if (n == 1 && takes(e[0])) even = plan_even(s, e[0], total, groups);
    for (int block = 0; block < groups; ++block) {
      if (even.splits) {
        const int w = plan_even_number(block, groups);
        CHECK(w >= 0 && w < groups && numbers.insert(w).second);
        int next = w / even.splits, parts = 0;
        PlanTask t;
        while (plan_even_take(s, e[0], even, w, groups, next, t)) {
          CHECK(arrived(Key(0, t.head, t.tile), w, t, plan_blocks(t.span)));
          CHECK(!t.cut || ++parts == 1);
        }
        continue;
      }
      PlanRun r;
      if (!plan_cut(s, total, groups, least, block, r)) continue;
      CHECK(numbers.insert(r.w).second && r.begin == r.w * r.per && r.end == std::min(total, r.begin + r.per));
      int i = 0;
      while (!(start[i] <= r.begin && takes(e[i]) && r.begin < start[i] + s.heads * plan_head_units(s, e[i]))) ++i;
      PlanPlace p = plan_find(s, e[i], i, start[i], r.begin - start[i]);
      PlanEntry at = e[i];
      int parts = 0;
      bool fine = true;
      for (bool more = true; more;) {
        int owner = -1;
        more = plan_take(
            s, r, at, p, [&](const PlanTask& t) {
              owner = p.entry;
              fine &= arrived(Key(owner, t.head, t.tile), r.w, t, plan_blocks(plan_span(s, e[owner], t.tile)));
              parts += t.cut;
            },
            [&](PlanPlace& q) {
              while (++q.entry < n)
                if (takes(at = e[q.entry])) return;
            });
        CHECK(more == (owner >= 0));
      }
      CHECK(fine && parts <= 2);
    }
    if (!even.splits && total) {
      // every run has a workgroup: their numbers are 0 .. with none left out
      CHECK(!numbers.empty() && *numbers.rbegin() + 1 == (int)numbers.size());
      const int64_t per = plan_per(s, total, groups, least);
      CHECK((int64_t)numbers.size() == (total + per - 1) / per);
    }
    if (even.splits) ++evens, rounds += even.tasks > groups;
    // every task's blocks once, its parts in the order of the workgroups, all arrived
    size_t tasks = 0;
    for (int i = 0; i < n; ++i) {
      if (!takes(e[i])) continue;
      for (int h = 0; h < s.heads; ++h)
        for (int t = 0; t < plan_tiles(s, e[i]); ++t) {
          const Key key(i, h, t);
          ++tasks;
          CHECK(got.count(key));
          auto mine = got[key];
          std::sort(mine.begin(), mine.end(), [](auto& a, auto& b) { return a.first < b.first; });
          int next = 0;
          for (size_t k = 0; k < mine.size(); ++k) {
            CHECK(mine[k].second.first == next);
            next = mine[k].second.end;
            CHECK(mine.size() == 1 || mine[k].first == ticket[key] + (int)k);
          }
          CHECK(next == plan_blocks(plan_span(s, e[i], t)));
          CHECK(mine.size() == 1 ? !count.count(key) : count[key] == (int)mine.size());
        }
    }
    CHECK(tasks == got.size());
  }
  if (evens < 50 || rounds < 5) { std::printf("%d even cuts, %d of more tasks than workgroups\\n", evens, rounds); return 1; }
}
"""


def test_every_workgroup_walks_its_run(tmp_path):
    """The functions that the kernels themselves call to number the runs and go from task to task (csrc/paged_plan.h), for
    whole launches: every task's blocks once, in parts whose places and tickets are their own and are all drawn."""
    (tmp_path / "walk.cpp").write_text(WALK)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'hawkpoint-npu-llm_amd' / 'csrc'}",
                    str(tmp_path / "walk.cpp"), "-o", str(tmp_path / "walk")], check=True)
    done = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
