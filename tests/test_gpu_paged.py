"""The paged KV cache on the GPU (include/hk_paged.h) against the float64 oracle.

Tolerances of the attention, per output o = sum_j p_j v_j (p the probabilities, A = sum_j p_j |v_j|):

- the result's rounding to bf16: 2^-8 |o| (half a step relative to the value, eps / 2)
- each probability's rounding to bf16 before its product: 2^-8 A
- a score's float32 error e_s moves p_j by e_s p_j relative, at most 2 e_s with the sum's share: 2 e_s A, where
  e_s <= D 2^-24 max|q||k| scale (a sum of D exact products, each partial sum rounded) + 2^-23 |s| for the scaling
- exp2 and the sum of the probabilities: a few 2^-23, below 2^-18 A for up to 8192 slots in runs

Inputs are drawn once; NaN in a place that a row does not see has to leave no trace at all."""

import ctypes

import numpy as np
import pytest

from _util import announce
from oracle import bf16
from oracle import paged as oracle

pytestmark = pytest.mark.gpu


def _bits(x):
    return bf16.to_bits(np.asarray(x, np.float32))


def _floats(bits):
    return bf16.from_bits(bits).astype(np.float64)


class Cache:
    """The oracle's cache and the same on the GPU."""

    def __init__(self, rng, *, layers=1, pages, kv_heads, page, dim, seqs, width, e4m3=False, gap=0, poison=True):
        from runtime import hip, paged

        self.e4m3, self.dim, self.page = e4m3, dim, page
        shape = (layers, pages, kv_heads, page, dim)
        self.scale = {x: rng.uniform(0.01, 0.03, (layers, kv_heads)).astype(np.float32) for x in "kv"}
        self.o = {"table": np.full((seqs, width), -1, np.int32), "length": np.zeros(seqs, np.int32),
                  "refs": np.zeros(pages, np.int32)}
        # every slot starts as NaN: whatever is read without having been written shows
        start = np.full(shape, np.nan if poison else 0.0)
        self.o["k"], self.o["v"] = start, start.copy()
        self.stride = kv_heads * page * dim + gap
        self.c = paged.PagedCache(layers=layers, kv_heads=kv_heads, head_dim=dim, page_size=page, pages=pages, seqs=seqs,
                                  table_width=width, dtype=paged.E4M3 if e4m3 else paged.BF16,
                                  page_stride=self.stride, layer_stride=pages * self.stride + gap)
        self.bufs = {"workspace": hip.DeviceBuffer(paged.WORKSPACE)}
        self.bufs["workspace"].zero()
        self.upload()
        if e4m3:
            for x in "kv":
                self.bufs[x + "_scale"] = hip.DeviceBuffer.from_array(self.scale[x])
                setattr(self.c, x + "_scale", self.bufs[x + "_scale"].ptr)

    def encode(self, x, which, layer):
        """Rows [.., kv heads, .., dim] as the pool's numbers; ``x`` has the heads on axis 1."""
        if not self.e4m3:
            return _bits(x)
        s = self.scale[which][layer].reshape(1, -1, 1, 1)
        return oracle.e4m3(np.asarray(x, np.float32) / s)

    def decode(self, codes, which, layer):
        if not self.e4m3:
            return _floats(codes)
        return oracle.from_e4m3(codes) * self.scale[which][layer].astype(np.float64).reshape(1, -1, 1, 1)

    def store(self, layer):
        """The oracle's rounding of appended rows."""
        def f(rows, which):
            x = np.asarray(rows)[None, :, None, :]
            return self.decode(self.encode(x.astype(np.float32), which, layer), which, layer)[0, :, 0]
        return f

    def _pool(self, which):
        layers, pages = self.o["k"].shape[:2]
        kind = np.uint8 if self.e4m3 else np.uint16
        flat = np.full(layers * self.c.layer_stride, 0x7F if self.e4m3 else 0x7FC0, kind)
        for l in range(layers):
            rows = flat[l * self.c.layer_stride:][:pages * self.stride].reshape(pages, self.stride)
            rows[:, :self.o["k"][l, 0].size] = self.encode(self.o[which][l], which, l).reshape(pages, -1)
        return flat

    def upload(self):
        from runtime import hip

        for x in ("k", "v", "table", "length", "refs"):
            if x in self.bufs:
                self.bufs[x].free()
            self.bufs[x] = hip.DeviceBuffer.from_array(self._pool(x) if x in "kv" else self.o[x])
            setattr(self.c, x, self.bufs[x].ptr)

    def download(self, which, layer):
        layers, pages, heads, page, dim = self.o["k"].shape
        flat = self.bufs[which].read(np.uint8 if self.e4m3 else np.uint16, layers * self.c.layer_stride)
        rows = flat[layer * self.c.layer_stride:][:pages * self.stride].reshape(pages, self.stride)
        return rows[:, :heads * page * dim].reshape(pages, heads, page, dim)

    def fill(self, rng, layer=0):
        """Normal keys and values, as the pool holds them, in the slots below each length; all others stay."""
        for s, n in enumerate(self.o["length"]):
            slot, page, at = oracle.slots_of(self.o, s, oracle.length_of(self.o, s))
            for x in "kv":
                new = rng.normal(size=(1, self.o["k"].shape[2], len(slot), self.dim)).astype(np.float32)
                got = self.decode(self.encode(new, x, layer), x, layer)[0]
                self.o[x][layer, page, :, at] = got.transpose(1, 0, 2)

    def give(self, lengths, rng):
        """Pages in a random order to sequences of these lengths."""
        free = list(rng.permutation(np.flatnonzero(self.o["refs"] == 0)))
        for s, n in enumerate(lengths):
            for j in range(-(-n // self.page)):
                self.o["table"][s, j] = free.pop()
                self.o["refs"][self.o["table"][s, j]] = 1
            self.o["length"][s] = n


def _dev(array):
    from runtime import hip

    return hip.DeviceBuffer.from_array(np.ascontiguousarray(array))


def _sync():
    from runtime import hip

    hip.check(hip.lib().hk_stream_sync(None), "sync")


def attention(cache, layer, q_bits, seqs, first, *, scale, window=0, max_new=None, stride=None, want_lse=True,
              stream=None):
    """(out [tokens, heads, dim] float64, lse, raw out bits): memory of rows that the call leaves alone reads as the
    pattern 0x4242."""
    from runtime import hip, paged

    tokens, heads, dim = q_bits.shape
    width = heads * dim
    stride = stride or width
    q = np.full((tokens + 1, stride), 0x7FC0, np.uint16)
    q[:tokens, :width] = q_bits.reshape(tokens, width)
    Q, S, F = _dev(q), _dev(np.asarray(seqs, np.int32)), _dev(np.asarray(first, np.int32))
    O, L = _dev(np.full((tokens + 1, stride), 0x4242, np.uint16)), _dev(np.full((tokens, heads), 77, np.float32))
    if max_new is None:
        max_new = max(1, int(np.diff(first).max(initial=1)))
    hip.check(paged.lib().hk_paged_attention(
        ctypes.byref(cache.c), layer, Q.ptr, stride, S.ptr, F.ptr, len(seqs), tokens, max_new, heads, scale, window, O.ptr,
        stride, L.ptr if want_lse else None, cache.bufs["workspace"].ptr, stream), "hk_paged_attention")
    hip.check(hip.lib().hk_stream_sync(stream), "sync")
    raw = O.read(np.uint16, (tokens + 1) * stride).reshape(tokens + 1, stride)
    assert np.all(raw[tokens] == 0x4242) and np.all(raw[:, width:] == 0x4242), "written outside the rows"
    raw = raw[:tokens, :width].reshape(tokens, heads, dim)
    return _floats(raw), L.read(np.float32, tokens * heads).reshape(tokens, heads), raw


def check_attention(got, lse, raw, want, q, cache, scale):
    out, want_lse, spread = want
    mine = spread[:, :, 0] != -1
    assert np.all(raw[~mine] == 0x4242), "rows of no entry were written"
    assert np.all(lse[~mine] == 77)
    dim = q.shape[2]
    k = cache.o["k"]
    top_k = np.abs(np.where(np.isfinite(k), k, 0)).max() * np.sqrt(dim)
    e_s = dim * 2.0**-24 * np.linalg.norm(q, axis=-1)[mine] * top_k * scale * 1.01 + 2.0**-23 * 64
    tol = 2.0**-8 * (np.abs(out[mine]) + spread[mine]) + (2 * e_s[:, None] + 2.0**-18) * spread[mine] + 1e-30
    nan = np.isnan(out[mine])
    np.testing.assert_array_equal(np.isnan(got[mine]), nan)
    err = np.where(nan, 0, np.abs(got[mine] - out[mine]))
    assert np.all((err <= tol) | nan), f"{(err > tol).sum()} outside, worst {np.nanmax(err / tol):.2f} of the tolerance"
    fine = np.isfinite(want_lse[mine])
    np.testing.assert_array_equal(lse[mine][~fine], want_lse[mine][~fine])
    off = np.abs(lse[mine][fine] - want_lse[mine][fine])
    assert np.all(off <= e_s[fine] + 2.0**-18 + 2.0**-22 * np.abs(want_lse[mine][fine])), off.max()


# (name, q heads, kv heads, dim, page, e4m3, [(length, new rows)], window)
CASES = [
    ("one token", 14, 2, 64, 16, False, [(1, 1)], 0),
    ("one token, 71 slots", 14, 2, 64, 16, False, [(71, 1)], 0),
    ("tokens at the edges of pages and tiles", 9, 3, 64, 16, False,
     [(n, 1) for n in (15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 255, 257)], 0),
    ("the same, 128 wide", 4, 1, 128, 32, False, [(n, 1) for n in (1, 31, 32, 33, 63, 64, 65, 127, 129, 300)], 0),
    ("the same, e4m3", 8, 2, 64, 64, True, [(n, 1) for n in (1, 32, 63, 64, 65, 128, 129, 300)], 0),
    ("the same, e4m3, 128 wide", 28, 4, 128, 16, True, [(n, 1) for n in (2, 47, 64, 130, 257)], 0),
    ("one head per kv head", 3, 3, 128, 128, False, [(40, 1), (400, 1)], 0),
    ("sixteen heads per kv head", 16, 1, 64, 256, False, [(40, 1), (700, 1)], 0),
    ("forty heads per kv head", 40, 1, 64, 16, False, [(33, 1), (150, 2)], 0),
    ("a long one and its split", 4, 2, 128, 16, False, [(5000, 1)], 0),
    ("long and short", 6, 2, 64, 32, False, [(3000, 1), (1, 1), (7, 1), (2500, 1)], 0),
    ("a few new tokens", 7, 1, 64, 16, False, [(200, 5), (5, 5), (64, 3), (65, 4), (1000, 2)], 0),
    ("a few new tokens, e4m3", 8, 2, 128, 64, True, [(200, 5), (5, 5), (64, 3), (700, 8)], 0),
    ("a short prompt", 14, 2, 64, 16, False, [(40, 40)], 0),
    ("a prompt", 14, 2, 64, 64, False, [(333, 333)], 0),
    ("a piece of a prompt", 8, 2, 128, 32, False, [(900, 131)], 0),
    ("a piece of a prompt, e4m3", 4, 2, 128, 16, True, [(515, 150)], 0),
    ("a piece of a prompt, e4m3, 64 wide", 6, 2, 64, 16, True, [(515, 150)], 0),
    ("pieces beside tokens", 8, 2, 64, 16, False, [(300, 100), (50, 1), (129, 1), (64, 64), (700, 1)], 0),
    ("pieces beside tokens, 24 heads per kv head", 48, 2, 64, 16, False, [(300, 40), (50, 1), (129, 1), (64, 2), (700, 1)], 0),
    ("the same, 20 heads, 128 wide, a window", 20, 1, 128, 32, True, [(300, 40), (50, 1), (129, 3), (700, 1), (9, 9)], 90),
    ("pieces beside tokens, 128 wide", 6, 2, 128, 64, True, [(300, 100), (50, 1), (129, 1), (64, 64), (700, 1)], 0),
    ("window of one", 4, 2, 64, 16, False, [(100, 1), (30, 30)], 1),
    ("window inside a tile", 4, 2, 64, 16, False, [(100, 1), (300, 90), (20, 20)], 37),
    ("window over tiles", 8, 1, 128, 32, False, [(700, 1), (600, 100), (99, 20)], 200),
    ("window longer than the context", 4, 2, 64, 16, False, [(100, 1), (70, 40)], 1000),
]


@pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])
def test_attention(hk_lib, case):
    name, hq, hkv, dim, page, e4m3, entries, window = case
    announce(f"paged attention: {name}")
    rng = np.random.default_rng(sum(map(ord, name)))
    need = sum(-(-n // page) for n, _ in entries)
    cache = Cache(rng, pages=need + 3, kv_heads=hkv, page=page, dim=dim, seqs=len(entries) + 2,
                  width=max(-(-n // page) for n, _ in entries) + 1, e4m3=e4m3, gap=64)
    cache.give([n for n, _ in entries], rng)
    cache.fill(rng)
    cache.upload()
    seqs = list(range(len(entries)))
    # the first two rows and the last one are of no entry
    first = np.cumsum([2] + [c for _, c in entries])
    q = _bits(rng.normal(size=(first[-1] + 1, hq, dim)) * 1.5)
    scale = dim**-0.5
    got, lse, raw = attention(cache, 0, q, seqs, first, scale=scale, window=window, stride=hq * dim + 24)
    want = oracle.attention(cache.o, 0, _floats(q), seqs, first, scale, window)
    check_attention(got, lse, raw, want, _floats(q), cache, scale)
    # the same result whatever the caller says of the entries' rows, and once more from the same workspace
    again = attention(cache, 0, q, seqs, first, scale=scale, window=window, stride=hq * dim + 24, want_lse=False)
    np.testing.assert_array_equal(again[2], raw)
    for max_new in (1, 4, 1000):
        check_attention(*attention(cache, 0, q, seqs, first, scale=scale, window=window, max_new=max_new), want,
                        _floats(q), cache, scale)


def test_attention_of_odd_batches(hk_lib):
    """Entries without rows, of length 0, longer than their sequence, of no sequence, with missing pages; the same
    sequence in two entries; sequences in another order."""
    announce("paged attention: odd batches")
    rng = np.random.default_rng(5)
    cache = Cache(rng, pages=40, kv_heads=2, page=16, dim=64, seqs=7, width=9)
    cache.give([0, 3, 100, 130, 64, 50, 20], rng)
    cache.fill(rng)
    # missing: a page in the middle, the only page, ids past the pool
    cache.o["table"][3, 2] = -1
    cache.o["table"][6, :2] = (-7, 40)
    cache.o["table"][5, 1] = 1 << 30
    cache.upload()
    seqs = [3, 0, 1, -1, 7, 6, 2, 2, 5, 4, 1 << 30]
    counts = [20, 2, 5, 1, 3, 4, 1, 90, 3, 0, 2]
    first = np.cumsum([0] + counts)
    q = _bits(rng.normal(size=(first[-1] + 3, 6, 64)))
    for window in (0, 18, 40):
        for max_new in (None, 1):
            got = attention(cache, 0, q, seqs, first, scale=0.2, window=window, max_new=max_new)
            check_attention(*got, oracle.attention(cache.o, 0, _floats(q), seqs, first, 0.2, window), _floats(q),
                            cache, 0.2)
    # lengths and first rows beyond what there is
    cache.o["length"][:] = (-5, 3, 10**9, 130, 64, 50, 20)
    cache.o["table"][2, 7:] = -1
    cache.upload()
    first[-1] = 10**6
    first[0] = -3
    got = attention(cache, 0, q, seqs, first, scale=0.2, max_new=100)
    check_attention(*got, oracle.attention(cache.o, 0, _floats(q), seqs, first, 0.2), _floats(q), cache, 0.2)


@pytest.mark.parametrize("dim,e4m3,counts,window", [
    (64, False, (1, 1), 60), (64, False, (4, 7), 60), (128, False, (90, 70), 60), (128, True, (90, 1), 60),
    (64, True, (3, 130), 60), (64, False, (2, 3), 1500), (128, False, (100, 80), 1500), (128, True, (5, 90), 1500)])
def test_attention_ignores_what_a_row_does_not_see(hk_lib, dim, e4m3, counts, window):
    """NaN and infinities in keys and values of later tokens, of slots left of the window, and behind the last slot."""
    announce(f"paged attention: poisoned slots, dim {dim}, e4m3 {e4m3}, rows {counts}, window {window}")
    rng = np.random.default_rng(7)
    lengths = [200, 147] if window < 100 else [2000, 1700]
    cache = Cache(rng, pages=sum(lengths) // 32 + 4, kv_heads=1, page=32, dim=dim, seqs=2, width=lengths[0] // 32 + 1,
                  e4m3=e4m3)
    cache.give(lengths, rng)
    cache.fill(rng)
    bad = [np.nan] if e4m3 else [np.nan, np.inf, -np.inf]
    for s, c in enumerate(counts):
        n = cache.o["length"][s]
        spots = [n - c - window, 0]  # left of every row's window
        if c > 1:
            spots.append(n - 1)  # seen by the last row alone
        for i, j in enumerate(spots):
            page, at = cache.o["table"][s, j // 32], j % 32
            cache.o["k"][0, page, 0, at, i] = bad[i % len(bad)]
            cache.o["v"][0, page, 0, at, 3 + i] = bad[(i + 1) % len(bad)]
    cache.upload()
    first = np.cumsum([0] + list(counts))
    q = _bits(rng.normal(size=(first[-1], 5, dim)))
    got, lse, raw = attention(cache, 0, q, [0, 1], first, scale=0.1, window=window)
    last = [first[i + 1] - 1 for i in range(2) if counts[i] > 1]
    with np.errstate(invalid="ignore"):
        want = oracle.attention(cache.o, 0, _floats(q), [0, 1], first, 0.1, window)
    keep = np.ones(first[-1], bool)
    keep[last] = False
    for r in last:  # the rows that see the values show it
        assert np.any(np.isnan(want[0][r]))
        np.testing.assert_array_equal(np.isnan(got[r]), np.isnan(want[0][r]))
    check_attention(got[keep], lse[keep], raw[keep], tuple(w[keep] for w in want), _floats(q)[keep], cache, 0.1)


def test_attention_of_a_poisoned_long_sequence(hk_lib):
    """One entry whose tiles are split over workgroups: the note of a NaN that only the last row sees comes with the
    parts."""
    announce("paged attention: poisoned slots of a sequence that is split")
    rng = np.random.default_rng(14)
    cache = Cache(rng, pages=160, kv_heads=2, page=16, dim=128, seqs=1, width=160)
    cache.give([2400], rng)
    cache.fill(rng)
    page = cache.o["table"][0, 2399 // 16]
    cache.o["v"][0, page, 1, 2399 % 16, 9] = np.nan
    cache.upload()
    q = _bits(rng.normal(size=(70, 4, 128)))
    want = oracle.attention(cache.o, 0, _floats(q), [0], [0, 70], 0.1)
    got = attention(cache, 0, q, [0], [0, 70], scale=0.1)
    assert np.isnan(want[0]).sum() == 2  # the last row's two heads of the second kv head
    check_attention(*got, want, _floats(q), cache, 0.1)


@pytest.mark.parametrize("dim,e4m3,entries", [
    (64, False, [(2500, 150)]), (128, False, [(3000, 90)]), (128, True, [(2600, 200)]), (64, True, [(1700, 300)]),
    (128, False, [(700, 700)]), (64, False, [(1500, 40), (1500, 41)])])
def test_attention_of_long_pieces(hk_lib, dim, e4m3, entries):
    """Tiles cut into equal parts, and into runs."""
    announce(f"paged attention: long pieces, dim {dim}, e4m3 {e4m3}, {entries}")
    rng = np.random.default_rng(dim + len(entries))
    need = sum(-(-n // 32) for n, _ in entries)
    cache = Cache(rng, layers=2, pages=need + 2, kv_heads=2, page=32, dim=dim, seqs=len(entries), width=need, e4m3=e4m3)
    cache.give([n for n, _ in entries], rng)
    for layer in (0, 1):
        cache.fill(rng, layer)
    cache.upload()
    first = np.cumsum([0] + [c for _, c in entries])
    q = _bits(rng.normal(size=(first[-1], 6, dim)))
    for layer in (0, 1):
        got = attention(cache, layer, q, range(len(entries)), first, scale=0.1)
        want = oracle.attention(cache.o, layer, _floats(q), range(len(entries)), first, 0.1)
        check_attention(*got, want, _floats(q), cache, 0.1)


def test_attention_of_more_tasks_than_workgroups(hk_lib):
    """32 kv heads of 25 tiles: whole tasks dealt out in rounds; with a second, empty entry, equal runs."""
    announce("paged attention: 800 tasks")
    rng = np.random.default_rng(31)
    cache = Cache(rng, pages=80, kv_heads=32, page=16, dim=64, seqs=2, width=80)
    cache.give([1200], rng)
    cache.fill(rng)
    cache.upload()
    q = _bits(rng.normal(size=(800, 128, 64)))
    calls = [attention(cache, 0, q, [0], [0, 800], scale=0.125), attention(cache, 0, q, [0, 1], [0, 800, 800], scale=0.125)]
    for g in (0, 17, 31):
        part = dict(cache.o, k=cache.o["k"][:, :, g:g + 1], v=cache.o["v"][:, :, g:g + 1])
        mine = slice(4 * g, 4 * g + 4)
        rows = np.arange(0, 800, 7)
        # (the oracle goes row by row: a seventh of them, each an entry of its own length)
        want = [np.concatenate(w) for w in zip(*(
            oracle.attention(dict(part, length=np.array([401 + t, 0], np.int32)), 0, _floats(q[t:t + 1, mine]), [0], [0, 1],
                             0.125) for t in rows))]
        for out, lse, raw in calls:
            check_attention(out[rows][:, mine], lse[rows][:, mine], raw[rows][:, mine], want, _floats(q[rows][:, mine]), cache,
                            0.125)


@pytest.mark.parametrize("n,counts", [(257, (1, 1, 1)), (700, (0, 1, 2)), (700, (1, 40, 0)), (4096, (1, 0, 1))])
def test_attention_of_many_entries(hk_lib, n, counts):
    """More entries than a workgroup has threads; sequences in any order, some in several entries."""
    announce(f"paged attention: {n} entries")
    rng = np.random.default_rng(n)
    cache = Cache(rng, pages=120, kv_heads=1, page=16, dim=64, seqs=40, width=4)
    cache.give(list(rng.integers(1, 49, 40)), rng)
    cache.fill(rng)
    cache.upload()
    seqs = rng.integers(0, 40, n)
    per = [counts[i % 3] for i in range(n)]
    first = np.cumsum([0] + per)
    q = _bits(rng.normal(size=(first[-1], 2, 64)))
    got = attention(cache, 0, q, seqs, first, scale=0.125)
    rows = np.unique(rng.integers(0, first[-1], 400))
    want = oracle.attention(cache.o, 0, _floats(q), seqs, first, 0.125)
    check_attention(*(x[rows] for x in got), tuple(w[rows] for w in want), _floats(q)[rows], cache, 0.125)


@pytest.mark.parametrize("heads,kv_heads,rows", [(4096, 1, 1), (4096, 1024, 1), (1024, 1024, 3), (96, 1, 2)])
def test_attention_of_many_heads(hk_lib, heads, kv_heads, rows):
    announce(f"paged attention: {heads} heads on {kv_heads}")
    rng = np.random.default_rng(heads + kv_heads)
    cache = Cache(rng, pages=12, kv_heads=kv_heads, page=16, dim=64, seqs=2, width=6)
    cache.give([70, 33], rng)
    cache.fill(rng)
    cache.upload()
    first = [0, rows, 2 * rows]
    q = _bits(rng.normal(size=(2 * rows, heads, 64)))
    got = attention(cache, 0, q, [1, 0], first, scale=0.125)
    check_attention(*got, oracle.attention(cache.o, 0, _floats(q), [1, 0], first, 0.125), _floats(q), cache, 0.125)


@pytest.mark.parametrize("e4m3,counts", [(True, (1, 3)), (True, (90, 40)), (False, (1, 1))])
def test_attention_with_the_smallest_scale(hk_lib, e4m3, counts):
    """A scale whose product with k_scale underflows: the mean of the values that a row sees, and of no others."""
    announce(f"paged attention: smallest scale, e4m3 {e4m3}, rows {counts}")
    rng = np.random.default_rng(12)
    cache = Cache(rng, pages=20, kv_heads=1, page=16, dim=64, seqs=2, width=10, e4m3=e4m3)
    cache.give([150, 77], rng)
    cache.fill(rng)
    cache.upload()
    first = np.cumsum([0] + list(counts))
    q = _bits(rng.normal(size=(first[-1], 3, 64)))
    got = attention(cache, 0, q, [0, 1], first, scale=1e-45, window=70)
    check_attention(*got, oracle.attention(cache.o, 0, _floats(q), [0, 1], first, 1e-45, 70), _floats(q), cache, 1e-45)


@pytest.mark.parametrize("dim,e4m3,counts", [(64, False, (1, 2)), (128, True, (1, 1)), (64, True, (90, 40)), (128, False, (90, 1))])
def test_attention_with_the_largest_scale(hk_lib, dim, e4m3, counts):
    """A scale whose product with log2 e overflows: queries of zeros score 0 everywhere, so their rows are the mean of the
    values that they see."""
    announce(f"paged attention: largest scale, dim {dim}, e4m3 {e4m3}, rows {counts}")
    rng = np.random.default_rng(13)
    cache = Cache(rng, pages=20, kv_heads=1, page=16, dim=dim, seqs=2, width=10, e4m3=e4m3)
    cache.scale = {x: np.full((1, 1), 2.0, np.float32) for x in "kv"}  # (the keys' scale adds to it)
    if e4m3:
        for x in "kv":
            cache.bufs[x + "_scale"].write(cache.scale[x])
    cache.give([150, 77], rng)
    cache.fill(rng)
    cache.upload()
    first = np.cumsum([0] + list(counts))
    q = np.zeros((first[-1], 3, dim), np.uint16)
    got = attention(cache, 0, q, [0, 1], first, scale=3e38, window=70)
    # (the oracle's scale does not matter to products of 0, and the tolerance's is that of the same products)
    check_attention(*got, oracle.attention(cache.o, 0, _floats(q), [0, 1], first, 1.0, 70), _floats(q), cache, 1.0)


@pytest.mark.parametrize("dim,e4m3,counts,lengths", [
    (64, False, (1, 1, 1), (4000, 30, 1)), (128, False, (200, 1, 60), (2000, 300, 61)), (128, True, (120,), (3500,)),
    (64, False, (40, 3, 0), (900, 2500, 5))])
def test_attention_in_place(hk_lib, dim, e4m3, counts, lengths):
    """The results in the queries' memory, of whole and of split tasks: the same bits as beside them."""
    from runtime import hip, paged

    announce(f"paged attention: in place, dim {dim}, {counts}")
    rng = np.random.default_rng(61)
    need = sum(-(-n // 16) for n in lengths)
    cache = Cache(rng, pages=need, kv_heads=2, page=16, dim=dim, seqs=len(counts), width=need, e4m3=e4m3)
    cache.give(list(lengths), rng)
    cache.fill(rng)
    cache.upload()
    first = np.cumsum([0] + list(counts))
    q = _bits(rng.normal(size=(first[-1], 8, dim)))
    want = attention(cache, 0, q, range(len(counts)), first, scale=0.1)[2]
    Q, F = _dev(q), _dev(first.astype(np.int32))
    hip.check(paged.lib().hk_paged_attention(
        ctypes.byref(cache.c), 0, Q.ptr, 8 * dim, None, F.ptr, len(counts), first[-1], max(counts), 8, 0.1, 0, Q.ptr,
        8 * dim, None, cache.bufs["workspace"].ptr, None), "hk_paged_attention")
    _sync()
    np.testing.assert_array_equal(Q.read(np.uint16, q.size).reshape(q.shape), want)


def test_attention_on_two_streams(hk_lib):
    """Calls in flight at once on streams of their own, each with its workspace; then the same stream after stream."""
    from runtime import hip, paged

    announce("paged attention: two streams")
    rng = np.random.default_rng(41)
    streams, sides = [], []
    for i in range(2):
        handle = ctypes.c_void_p()
        hip.check(hk_lib.hk_stream_create(ctypes.byref(handle)), "hk_stream_create")
        streams.append(handle.value)
        cache = Cache(rng, pages=400, kv_heads=2, page=16, dim=64, seqs=3, width=200)
        cache.give([3000, 1500, 200], rng)
        cache.fill(rng)
        cache.upload()
        first = np.array([0, 1, 2, 3 + 90 * i])
        q = _bits(rng.normal(size=(first[-1], 4, 64)))
        sides.append((cache, q, first, oracle.attention(cache.o, 0, _floats(q), [0, 1, 2], first, 0.125)))
    bufs = []
    for cache, q, first, _ in sides:
        bufs.append((_dev(q), _dev(first.astype(np.int32)), _dev(np.zeros(q.shape, np.uint16)),
                     _dev(np.zeros(q.shape[:2], np.float32))))
    _sync()
    for _ in range(20):
        for stream, (cache, q, first, _), (Q, F, O, L) in zip(streams, sides, bufs):
            hip.check(paged.lib().hk_paged_attention(
                ctypes.byref(cache.c), 0, Q.ptr, 256, None, F.ptr, 3, len(q), int(np.diff(first).max()), 4, 0.125, 0, O.ptr, 256,
                L.ptr, cache.bufs["workspace"].ptr, stream), "hk_paged_attention")
    for stream, (cache, q, first, want), (Q, F, O, L) in zip(streams, sides, bufs):
        hip.check(hk_lib.hk_stream_sync(stream), "sync")
        raw = O.read(np.uint16, q.size).reshape(q.shape)
        check_attention(_floats(raw), L.read(np.float32, q[:, :, 0].size).reshape(q.shape[:2]), raw, want, _floats(q), cache, 0.125)
    for stream in streams:
        hip.check(hk_lib.hk_stream_destroy(stream), "hk_stream_destroy")


def test_attention_layers_and_far_pages(hk_lib):
    """Layers of their own, and pages more than 4 GiB into the pool."""
    from runtime import hip

    announce("paged attention: pages beyond 32-bit offsets")
    rng = np.random.default_rng(8)
    cache = Cache(rng, layers=2, pages=6, kv_heads=1, page=16, dim=64, seqs=1, width=4, poison=False)
    cache.give([50], rng)
    for layer in (0, 1):
        cache.fill(rng, layer)
    cache.upload()
    q = _bits(rng.normal(size=(2, 2, 64)))
    for layer in (0, 1):
        got = attention(cache, layer, q, [0], [0, 2], scale=0.125)
        check_attention(*got, oracle.attention(cache.o, layer, _floats(q), [0], [0, 2], 0.125), _floats(q), cache,
                        0.125)
    # the same pages 1 GiB of elements apart: page 5 starts 10 GiB into a pool
    stride = 1 << 30
    far = {x: hip.DeviceBuffer(2 * (5 * stride + 16 * 64)) for x in "kv"}
    for x in "kv":
        rows = cache.encode(cache.o[x][1], x, 1)
        for p in range(6):
            far[x].write(rows[p], 2 * p * stride)
        setattr(cache.c, x, far[x].ptr)
    cache.c.page_stride, cache.c.layer_stride, cache.c.layers = stride, 6 * stride, 1
    got = attention(cache, 0, q, [0], [0, 2], scale=0.125)
    check_attention(*got, oracle.attention(cache.o, 1, _floats(q), [0], [0, 2], 0.125), _floats(q), cache, 0.125)


# ---- append ----


def _tables(slots, dim, rng):
    angle = np.arange(slots)[:, None] * 10000.0 ** (-np.arange(dim // 2) / (dim // 2))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


@pytest.mark.parametrize("hq,hkv,dim,page,e4m3,rope", [(14, 2, 64, 16, False, True), (9, 3, 64, 32, True, True),
                                                       (8, 2, 128, 16, False, False), (28, 4, 128, 64, True, True)])
def test_append(hk_lib, hq, hkv, dim, page, e4m3, rope):
    """bf16: the numbers are one rounding of float32 a cos - b sin (half a step, 2^-8 relative to the result, after
    products and a difference each rounded by 2^-24 of their operands); values are stored as they are.  e4m3: the
    nearest code of x / scale, or its neighbour where float32 falls on the other side of a border."""
    from runtime import hip, paged

    announce(f"paged append: {hq}/{hkv} heads of {dim}, page {page}, e4m3 {e4m3}")
    rng = np.random.default_rng(dim + page)
    # a new sequence, one token, over a page's end, no rows, more rows than tokens, of no sequence
    entries = [(0, 37, 37), (1, 50, 1), (2, page + 3, 9), (3, 20, 0), (4, 2, 5), (9, 0, 2)]
    cache = Cache(rng, layers=2, pages=30, kv_heads=hkv, page=page, dim=dim, seqs=5, width=6, e4m3=e4m3, gap=32)
    cache.give([n for _, n, _ in entries[:5]], rng)
    for layer in (0, 1):
        cache.fill(rng, layer)
    cache.o["table"][2, 1] = -1  # where some of the rows would go
    cache.upload()
    untouched = [[cache.download(x, l).copy() for x in "kv"] for l in (0, 1)]
    first = np.cumsum([1] + [c for _, _, c in entries])
    tokens, stride = int(first[-1]) + 2, (hq + 2 * hkv) * dim + 16
    qkv = np.full((tokens, stride), 0x7FC0, np.uint16)
    x = _bits(rng.normal(size=(tokens, hq + 2 * hkv, dim)) * 3)
    qkv[:, :-16] = x.reshape(tokens, -1)
    if e4m3:  # saturation, and NaN which stays one
        x[first[1], hq, 5] = _bits([1e6])[0]
        x[first[1], hq + hkv, 6] = _bits([-1e6])[0]
        x[first[1], hq + hkv, 7] = 0x7FC0
        qkv[:, :-16] = x.reshape(tokens, -1)
    cos, sin = _tables(6 * page, dim, rng) if rope else (None, None)
    C, S = (None if t is None else _dev(t) for t in (cos, sin))
    IN, OUT = _dev(qkv), _dev(np.full((tokens, hq * dim + 8), 0x4242, np.uint16))
    SEQ, FIRST = _dev(np.array([s for s, _, _ in entries], np.int32)), _dev(first.astype(np.int32))

    def call(q_out, q_stride):
        hip.check(paged.lib().hk_paged_append(
            ctypes.byref(cache.c), 1, IN.ptr, stride, C and C.ptr, S and S.ptr, 6 * page, SEQ.ptr, FIRST.ptr, len(entries),
            tokens, hq, q_out, q_stride, None), "hk_paged_append")
        _sync()

    call(OUT.ptr, hq * dim + 8)
    before = {y: cache.o[y].copy() for y in "kv"}
    want = oracle.append(cache.o, 1, _floats(x), [s for s, _, _ in entries], first, hq, cos, sin, cache.store(1))
    raw = OUT.read(np.uint16, tokens * (hq * dim + 8)).reshape(tokens, -1)
    assert np.all(raw[:, hq * dim:] == 0x4242)
    raw = raw[:, :hq * dim].reshape(tokens, hq, dim)
    mine = ~np.isnan(want[:, 0, 0])
    assert np.all(raw[~mine] == 0x4242)
    f = np.abs(_floats(x)[:, :hq])
    a = f + np.roll(f, dim // 2, -1)
    assert np.all(np.abs(_floats(raw)[mine] - want[mine]) <= 2.0**-8 * np.abs(want[mine]) + 2.0**-23 * a[mine])
    for y, i in (("k", 0), ("v", 1)):
        got = cache.download(y, 1)
        written = ~((cache.o[y][1] == before[y][1]) | (np.isnan(cache.o[y][1]) & np.isnan(before[y][1])))
        np.testing.assert_array_equal(got[~written], untouched[1][i][~written])
        want_codes = cache.encode(cache.o[y][1], y, 1)
        step = np.abs(got[written].astype(int) - want_codes[written].astype(int))
        if e4m3:  # (a NaN's sign says nothing)
            step[(got[written] & 0x7F == 0x7F) & (want_codes[written] == 0x7F)] = 0
        assert step.max() <= 1 and (step == 0).mean() > 0.99 and (y == "k" or step.max() == 0)
        np.testing.assert_array_equal(cache.download(y, 0), untouched[0][i])
    # in place, and without queries
    call(IN.ptr, stride)
    back = IN.read(np.uint16, tokens * stride).reshape(tokens, stride)
    np.testing.assert_array_equal(back[:, :hq * dim].reshape(raw.shape)[mine], raw[mine])
    np.testing.assert_array_equal(back[:, hq * dim:], qkv[:, hq * dim:])
    once = [cache.download(y, 1) for y in "kv"]
    call(None, 0)
    for y, was in zip("kv", once):
        np.testing.assert_array_equal(cache.download(y, 1), was)


def test_append_is_the_decode_steps_append(hk_lib):
    """The rows that hk_attention_decode puts into its contiguous cache, bit for bit, and its attention's numbers."""
    from runtime import hip
    from runtime.qwen_engine import rope_tables

    announce("paged append and attention against hk_attention_decode")
    rng = np.random.default_rng(11)
    hq, hkv, ctx, p = 14, 2, 512, 300
    cos, sin = rope_tables(1e6, 64, ctx)
    kc, vc = (np.zeros((hkv, ctx, 64), np.uint16) for _ in range(2))
    kc[:, :p], vc[:, :p] = (_bits(rng.normal(size=(hkv, p, 64))) for _ in range(2))
    qkv = _bits(rng.normal(size=(hq + 2 * hkv) * 64))
    QKV, COS, SIN, KC, VC = map(_dev, (qkv, cos, sin, kc, vc))
    OUT = hip.DeviceBuffer(2 * hq * 64)
    hip.check(hk_lib.hk_attention_decode(QKV.ptr, COS.ptr, SIN.ptr, KC.ptr, VC.ptr, p, ctx, hq, hkv, 64, OUT.ptr, None),
              "hk_attention_decode")
    _sync()
    want = OUT.read(np.uint16, hq * 64)
    from runtime import paged

    cache = Cache(rng, pages=40, kv_heads=hkv, page=16, dim=64, seqs=1, width=32)
    cache.give([p + 1], rng)
    slot, page, at = oracle.slots_of(cache.o, 0, p)
    for x, rows in (("k", kc), ("v", vc)):
        cache.o[x][0, page, :, at] = _floats(rows[:, :p]).transpose(1, 0, 2)
    cache.upload()
    SEQ, FIRST, Q = _dev(np.zeros(1, np.int32)), _dev(np.array([0, 1], np.int32)), hip.DeviceBuffer(2 * hq * 64)
    hip.check(paged.lib().hk_paged_append(ctypes.byref(cache.c), 0, QKV.ptr, (hq + 2 * hkv) * 64, COS.ptr, SIN.ptr, ctx,
                                          None, FIRST.ptr, 1, 1, hq, Q.ptr, hq * 64, None), "hk_paged_append")
    _sync()
    for x, ref in (("k", KC), ("v", VC)):
        held = ref.read(np.uint16, hkv * ctx * 64).reshape(hkv, ctx, 64)[:, p]
        np.testing.assert_array_equal(cache.download(x, 0)[cache.o["table"][0, p // 16], :, p % 16], held)
        cache.o[x][0, cache.o["table"][0, p // 16], :, p % 16] = _floats(held)
    q = Q.read(np.uint16, hq * 64).reshape(1, hq, 64)
    got = attention(cache, 0, q, [0], [0, 1], scale=0.125)
    ref = oracle.attention(cache.o, 0, _floats(q), [0], [0, 1], 0.125)
    check_attention(*got, ref, _floats(q), cache, 0.125)
    # both within their tolerance of float64: a bf16 step of each other and the probabilities' rounding
    assert np.all(np.abs(_floats(want).reshape(1, hq, 64) - got[0]) <= 2.0**-7 * np.abs(ref[0]) + 2.0**-8 * ref[2] * 1.1)


# ---- fork and compaction ----


def fork(cache, child, parent, keep, grow):
    """Both forks; the status words."""
    from runtime import hip, paged

    arrays = [None if a is None else _dev(np.asarray(a, np.int32)) for a in (child, parent, keep, grow)]
    S = _dev(np.full(2, -9, np.int32))
    n = len(next(a for a in (child, parent, keep, grow) if a is not None))
    hip.check(paged.lib().hk_paged_fork(ctypes.byref(cache.c), *(a and a.ptr for a in arrays), n, S.ptr,
                                        cache.bufs["workspace"].ptr, None), "hk_paged_fork")
    _sync()
    return tuple(S.read(np.int32, 2).tolist())


def same(cache):
    """The GPU's cache is the oracle's, all of it."""
    for x in ("table", "length", "refs"):
        np.testing.assert_array_equal(cache.bufs[x].read(np.int32, cache.o[x].size).reshape(cache.o[x].shape), cache.o[x],
                                      err_msg=x)
    for l in range(cache.o["k"].shape[0]):
        for x in "kv":
            np.testing.assert_array_equal(cache.download(x, l), cache.encode(cache.o[x][l], x, l), err_msg=x)


@pytest.mark.parametrize("page,dim,e4m3,seed", [(16, 64, False, 0), (32, 128, True, 1), (64, 64, True, 2)])
def test_fork_and_compact_in_random_order(hk_lib, page, dim, e4m3, seed):
    """A hundred random calls: new answers, reordered beams, tokens added and taken back, sequences freed, entries
    that are not valid, pools too full, compactions, each compared with the oracle's whole cache."""
    from runtime import hip, paged

    announce(f"paged fork: page {page}, dim {dim}, e4m3 {e4m3}")
    rng = np.random.default_rng(seed)
    seqs, width = 9, 6
    cache = Cache(rng, layers=2, pages=10, kv_heads=2, page=page, dim=dim, seqs=seqs, width=width, e4m3=e4m3, gap=16,
                  poison=False)
    outcomes = set()
    for step in range(100):
        n = int(rng.integers(1, seqs + 1))
        child = rng.permutation(seqs)[:n]
        kind = rng.integers(0, 6)
        length = cache.o["length"]
        if kind == 0:  # the next tokens
            parent, keep, grow = child, length[child], rng.integers(0, page, n)
        elif kind == 1:  # answers and beams
            parent = rng.integers(0, seqs, n)
            keep, grow = length[parent], rng.integers(0, 3, n)
        elif kind == 2:  # prefixes
            parent = rng.integers(0, seqs, n)
            keep, grow = rng.integers(0, length[parent] + 1), rng.integers(0, page, n)
        elif kind == 3:  # freeing
            parent, keep, grow = np.full(n, -1), np.zeros(n, int), np.zeros(n, int)
        elif kind == 4 and step % 3 == 0:  # not valid in one of several ways
            parent, keep, grow = child.copy(), length[child].copy(), np.ones(n, int)
            i = int(rng.integers(n))
            bad = rng.integers(0, 6)
            if bad == 0 and n > 1:
                child[i] = child[i - 1]
            elif bad == 1:
                child[i] = seqs
            elif bad == 2:
                keep[i] += 1
            elif bad == 3:
                parent[i], keep[i] = -1, 1
            elif bad == 4:
                grow[i] = width * page
            else:
                grow[i] = -1
        else:
            live = oracle.compact(cache.o)
            L = _dev(np.zeros(1, np.int32))
            hip.check(paged.lib().hk_paged_compact(ctypes.byref(cache.c), cache.c.table, cache.c.refs, L.ptr,
                                                   cache.bufs["workspace"].ptr, None), "hk_paged_compact")
            _sync()
            assert L.read(np.int32, 1)[0] == live
            same(cache)
            continue
        want = oracle.fork(cache.o, *(list(map(int, a)) for a in (child, parent, keep, grow)))
        assert fork(cache, child, parent, keep, grow) == want, (step, kind)
        outcomes.add(want[0])
        same(cache)
        if want[0] == 0 and rng.random() < 0.5:  # contents that tell the pages apart
            cache.fill(rng, int(rng.integers(2)))
            cache.upload()
    assert outcomes == {0, 1, 2}


def test_fork_defaults_and_aliases(hk_lib):
    """NULL arrays, and `keep` that is the cache's own lengths."""
    from runtime import hip, paged

    announce("paged fork: defaults")
    rng = np.random.default_rng(3)
    cache = Cache(rng, pages=12, kv_heads=1, page=16, dim=64, seqs=3, width=4, poison=False)
    cache.give([5, 16, 31], rng)
    cache.fill(rng)
    cache.upload()
    S, G = _dev(np.zeros(2, np.int32)), _dev(np.array([1, 1, 2], np.int32))
    for grow, keep in ((None, None), (G.ptr, None), (G.ptr, cache.c.length), (cache.c.length, cache.c.length)):
        hip.check(paged.lib().hk_paged_fork(ctypes.byref(cache.c), None, None, keep, grow, 3, S.ptr,
                                            cache.bufs["workspace"].ptr, None), "hk_paged_fork")
        _sync()
        n = cache.o["length"].tolist()
        add = [0] * 3 if grow is None else [1, 1, 2] if grow == G.ptr else n
        assert tuple(S.read(np.int32, 2)) == oracle.fork(cache.o, [0, 1, 2], [0, 1, 2], n, add)
        same(cache)


@pytest.mark.parametrize("pages,seqs", [(1, 1), (64, 5), (1500, 130), (5000, 1030)])
def test_fork_and_compact_sizes(hk_lib, pages, seqs):
    """Pools of more pages, and calls of more entries, than a workgroup has threads; compaction into other tables."""
    from runtime import hip, paged

    announce(f"paged fork: {pages} pages, {seqs} sequences")
    rng = np.random.default_rng(pages)
    width = max(1, pages // seqs - 1)
    cache = Cache(rng, pages=pages, kv_heads=1, page=16, dim=64, seqs=seqs, width=width, poison=False)
    grow = rng.integers(0, 16 * width + 1, seqs)
    zero = [0] * seqs
    assert fork(cache, None, None, zero, grow) == oracle.fork(cache.o, range(seqs), range(seqs), zero, grow) == (0, 0)
    cache.fill(rng)
    cache.upload()
    child = rng.permutation(seqs)
    parent = rng.integers(0, seqs, seqs)
    keep = [int(rng.integers(0, cache.o["length"][p] + 1)) for p in parent]
    assert fork(cache, child, parent, keep, zero) == oracle.fork(cache.o, child, parent, keep, zero) == (0, 0)
    same(cache)
    T, R, L = _dev(np.zeros_like(cache.o["table"])), _dev(np.zeros_like(cache.o["refs"])), _dev(np.zeros(1, np.int32))
    was = {x: cache.o[x].copy() for x in ("table", "refs")}
    hip.check(paged.lib().hk_paged_compact(ctypes.byref(cache.c), T.ptr, R.ptr, L.ptr, cache.bufs["workspace"].ptr, None),
              "hk_paged_compact")
    _sync()
    assert oracle.compact(cache.o) == L.read(np.int32, 1)[0]
    np.testing.assert_array_equal(T.read(np.int32, cache.o["table"].size), cache.o["table"].ravel())
    np.testing.assert_array_equal(R.read(np.int32, pages), cache.o["refs"])
    cache.o.update(was)
    same(cache)


def test_far_pages_are_written_copied_and_moved(hk_lib):
    """Pages 2 GiB apart: an append, a fork that copies slots and a compaction that moves pages more than 4 GiB away."""
    from runtime import hip, paged

    announce("paged cache: writes beyond 32-bit offsets")
    rng = np.random.default_rng(9)
    cache = Cache(rng, pages=6, kv_heads=1, page=16, dim=64, seqs=3, width=5, poison=False)
    cache.o["table"][0, 0], cache.o["table"][2, :4] = 5, [0, 1, 2, 3]
    cache.o["refs"][:] = (1, 1, 1, 1, 0, 1)
    cache.o["length"][:] = (10, 0, 60)
    cache.fill(rng)
    cache.upload()
    stride, size = 1 << 30, 16 * 64
    far = {x: hip.DeviceBuffer(2 * (5 * stride + size)) for x in "kv"}

    def put():
        for x in "kv":
            for p in range(6):
                far[x].write(cache.encode(cache.o[x][0], x, 0)[p], 2 * p * stride)

    def held():
        for x in "kv":
            want = cache.encode(cache.o[x][0], x, 0)
            for s in range(3):
                for j in range(int(cache.o["length"][s])):
                    p = int(cache.o["table"][s, j // 16])
                    got = far[x].read(np.uint16, size, 2 * p * stride).reshape(1, 16, 64)
                    np.testing.assert_array_equal(got[:, j % 16], want[p, :, j % 16])

    put()
    for x in "kv":
        setattr(cache.c, x, far[x].ptr)
    cache.c.page_stride = cache.c.layer_stride = stride
    step = ([0, 1], [0, 0], [10, 10], [1, 2])
    assert fork(cache, *step) == oracle.fork(cache.o, *step) == (0, 0)  # sequence 1 gets page 4
    assert cache.o["table"][1, 0] == 4
    held()
    x = _bits(rng.normal(size=(3, 4, 64)))
    IN, SEQS, FIRST = _dev(x), _dev(np.array([0, 1], np.int32)), _dev(np.array([0, 1, 3], np.int32))
    hip.check(paged.lib().hk_paged_append(ctypes.byref(cache.c), 0, IN.ptr, 256, None, None, 0, SEQS.ptr, FIRST.ptr, 2, 3, 2,
                                          None, 0, None), "hk_paged_append")
    _sync()
    oracle.append(cache.o, 0, _floats(x), [0, 1], [0, 1, 3], 2, None, None, lambda rows, which: rows)
    held()
    free = ([2], [2], [0], [0])
    assert fork(cache, *free) == oracle.fork(cache.o, *free) == (0, 0)
    LIVE = _dev(np.zeros(1, np.int32))
    hip.check(paged.lib().hk_paged_compact(ctypes.byref(cache.c), cache.c.table, cache.c.refs, LIVE.ptr,
                                           cache.bufs["workspace"].ptr, None), "hk_paged_compact")
    _sync()
    assert LIVE.read(np.int32, 1)[0] == oracle.compact(cache.o) == 2
    assert sorted(cache.o["table"][:2, 0]) == [0, 1]
    for name in ("table", "length", "refs"):
        np.testing.assert_array_equal(cache.bufs[name].read(np.int32, cache.o[name].size), cache.o[name].ravel())
    held()


# ---- together ----


class Graph:
    """A stream's work between ``with`` and its end, captured and replayed through the HIP runtime of libhk.so."""

    def __init__(self, stream):
        # the runtime that libhk.so is bound to is in the process already: its functions by their global names
        path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
        self.hip, self.stream = ctypes.CDLL(path), ctypes.c_void_p(stream)
        self.graph, self.exe = ctypes.c_void_p(), ctypes.c_void_p()

    def _ok(self, rc):
        assert rc == 0, rc

    def __enter__(self):
        self._ok(self.hip.hipStreamBeginCapture(self.stream, 0))

    def __exit__(self, kind, *_):
        self._ok(self.hip.hipStreamEndCapture(self.stream, ctypes.byref(self.graph)))
        if kind is None:
            self._ok(self.hip.hipGraphInstantiate(ctypes.byref(self.exe), self.graph, None, None, ctypes.c_size_t(0)))

    def replay(self):
        self._ok(self.hip.hipGraphLaunch(self.exe, self.stream))

    def close(self):
        self._ok(self.hip.hipGraphExecDestroy(self.exe))
        self._ok(self.hip.hipGraphDestroy(self.graph))


@pytest.mark.parametrize("dim,e4m3", [(64, False), (128, True)])
def test_a_captured_step_serves_every_later_length(hk_lib, dim, e4m3):
    """Fork, append and attention of one decode step in a graph: each replay goes on from the lengths that the one
    before left on the device, over page ends and past lengths that cut the work in other places, with eager calls and
    synchronisations between the replays."""
    from runtime import hip, paged

    announce(f"paged cache: captured step, dim {dim}, e4m3 {e4m3}")
    rng = np.random.default_rng(51)
    hq, hkv, page, seqs, width = 6, 2, 16, 3, 40
    cache = Cache(rng, pages=110, kv_heads=hkv, page=page, dim=dim, seqs=seqs, width=width, e4m3=e4m3, poison=False)
    cache.give([30, 599, 15], rng)
    cache.fill(rng)
    cache.upload()
    handle = ctypes.c_void_p()
    hip.check(hk_lib.hk_stream_create(ctypes.byref(handle)), "hk_stream_create")
    stream = handle.value
    cos, sin = _tables(width * page, dim, rng)
    C, S, ONE = _dev(cos), _dev(sin), _dev(np.ones(seqs, np.int32))
    FIRST, STATUS = _dev(np.arange(seqs + 1, dtype=np.int32)), _dev(np.zeros(2, np.int32))
    IN, Q = hip.DeviceBuffer(2 * seqs * (hq + 2 * hkv) * dim), hip.DeviceBuffer(2 * seqs * hq * dim)
    OUT, LSE = hip.DeviceBuffer(2 * seqs * hq * dim), hip.DeviceBuffer(4 * seqs * hq)
    _sync()
    lib, c, ws = paged.lib(), ctypes.byref(cache.c), cache.bufs["workspace"].ptr
    graph = Graph(stream)
    with graph:
        hip.check(lib.hk_paged_fork(c, None, None, None, ONE.ptr, seqs, STATUS.ptr, ws, stream), "hk_paged_fork")
        hip.check(lib.hk_paged_append(c, 0, IN.ptr, (hq + 2 * hkv) * dim, C.ptr, S.ptr, width * page, None, FIRST.ptr, seqs,
                                      seqs, hq, Q.ptr, hq * dim, stream), "hk_paged_append")
        hip.check(lib.hk_paged_attention(c, 0, Q.ptr, hq * dim, None, FIRST.ptr, seqs, seqs, 1, hq, dim**-0.5, 0, OUT.ptr,
                                         hq * dim, LSE.ptr, ws, stream), "hk_paged_attention")
    for step in range(6):
        x = _bits(rng.normal(size=(seqs, hq + 2 * hkv, dim)))
        IN.write(x)
        graph.replay()
        hip.check(hk_lib.hk_stream_sync(stream), "sync")
        n = [int(v) for v in cache.o["length"]]
        assert tuple(STATUS.read(np.int32, 2)) == oracle.fork(cache.o, [0, 1, 2], [0, 1, 2], n, [1] * 3) == (0, 0)
        oracle.append(cache.o, 0, _floats(x), [0, 1, 2], [0, 1, 2, 3], hq, cos, sin, cache.store(0))
        # (a key at a rounding border may be its neighbour: the attention is checked on what the pool holds)
        for y in "kv":
            cache.o[y][0] = cache.decode(cache.download(y, 0), y, 0)
        q = _floats(Q.read(np.uint16, seqs * hq * dim).reshape(seqs, hq, dim))
        raw = OUT.read(np.uint16, seqs * hq * dim).reshape(seqs, hq, dim)
        lse = LSE.read(np.float32, seqs * hq).reshape(seqs, hq)
        want = oracle.attention(cache.o, 0, q, [0, 1, 2], [0, 1, 2, 3], dim**-0.5)
        check_attention(_floats(raw), lse, raw, want, q, cache, dim**-0.5)
        # the eager call on the same inputs gives the same bits
        again = attention(cache, 0, _bits(q), [0, 1, 2], [0, 1, 2, 3], scale=dim**-0.5)
        np.testing.assert_array_equal(again[2], raw)
    graph.close()
    hip.check(hk_lib.hk_stream_destroy(stream), "hk_stream_destroy")


def test_chats_share_a_prompt(hk_lib):
    """As a server uses it: a prompt in two pieces, three answers forked from it, decode steps of all of them at once
    over two layers, one taken back, one freed, the pool compacted, and on.  Each attention against the oracle."""
    from runtime import paged

    announce("paged cache: chats that share a prompt")
    rng = np.random.default_rng(21)
    hq, hkv, dim, page, layers = 6, 2, 64, 16, 2
    kv = paged.PagedKV(layers=layers, kv_heads=hkv, head_dim=dim, page_size=page, pages=30, seqs=5, table_width=8)
    cos, sin = _tables(8 * page, dim, rng)
    C, S = _dev(cos), _dev(sin)
    o = {"k": np.zeros((layers, 30, hkv, page, dim)), "v": np.zeros((layers, 30, hkv, page, dim)),
         "table": np.full((5, 8), -1, np.int32), "length": np.zeros(5, np.int32), "refs": np.zeros(30, np.int32)}

    def forked(child, parent, keep, grow):
        assert oracle.fork(o, child, parent, keep, grow) == (0, 0)
        kv.fork(child, parent, keep, grow)
        for name in ("table", "length", "refs"):
            got = {"table": kv.table, "length": kv.lengths, "refs": kv.refs}[name]()
            np.testing.assert_array_equal(got, o[name])

    def stepped(seqs, counts):
        first = np.cumsum([0] + counts)
        for layer in range(layers):
            x = _bits(rng.normal(size=(first[-1], hq + 2 * hkv, dim)))
            IN, Q, OUT = _dev(x), _dev(np.zeros((first[-1], hq, dim), np.uint16)), _dev(np.zeros((first[-1], hq, dim),
                                                                                               np.uint16))
            kv.append(layer, IN.ptr, seqs, first, hq, rope=(C.ptr, S.ptr, 8 * page), q_out=Q.ptr)
            kv.attention(layer, Q.ptr, seqs, first, hq, OUT.ptr)
            _sync()
            oracle.append(o, layer, _floats(x), seqs, first, hq, cos, sin, lambda rows, which: _floats(_bits(rows)))
            # The float32 rotation may fall to the neighbouring bf16, 2^-7 of the smaller one at most (and where the
            # two products cancel, by 2^-22 of either): the attention is checked on what the pool holds.
            for y in "kv":
                pool = _floats(kv.bufs[y].read(np.uint16, kv.bufs[y].nbytes // 2).reshape(o[y].shape)[layer])
                mine = np.any(o[y][layer] != 0, axis=-1)  # slots that were written: the others hold anything
                was, got = o[y][layer][mine], pool[mine]
                assert np.all(np.abs(got - was) <= 2.0**-7 * np.abs(was) + 2.0**-20)
                o[y][layer][mine] = got
            q = _floats(Q.read(np.uint16, Q.nbytes // 2).reshape(-1, hq, dim))
            got = _floats(OUT.read(np.uint16, OUT.nbytes // 2).reshape(-1, hq, dim))
            want, _, spread = oracle.attention(o, layer, q, seqs, first, dim**-0.5)
            e_s = dim * 2.0**-24 * np.linalg.norm(q, axis=-1) * np.abs(o["k"]).max() * 1.01 + 2.0**-23 * 64
            tol = 2.0**-8 * (np.abs(want) + spread) + (2 * e_s[..., None] + 2.0**-18) * spread + 1e-30
            assert np.all(np.abs(got - want) <= tol)

    forked([0], [0], [0], [21])
    stepped([0], [21])
    forked([0], [0], [21], [30])
    stepped([0], [30])
    forked([1, 2, 3], [0, 0, 0], [51, 51, 40], [1, 1, 2])
    stepped([1, 2, 3], [1, 1, 2])
    for _ in range(14):
        n = [int(x) for x in o["length"]]
        forked([0, 1, 2, 3], [0, 1, 2, 3], n[:4], [1] * 4)
        stepped([2, 0, 1, 3], [1] * 4)
    n = [int(x) for x in o["length"]]
    forked([1, 2], [1, 2], [n[1] - 20, 0], [3, 0])  # taken back and corrected; freed
    stepped([1], [3])
    assert kv.compact() == oracle.compact(o)
    np.testing.assert_array_equal(kv.table(), o["table"])
    np.testing.assert_array_equal(kv.refs(), o["refs"])
    for _ in range(3):
        n = [int(x) for x in o["length"]]
        forked([0, 1, 3], [0, 1, 3], [n[0], n[1], n[3]], [1, 2, 1])
        stepped([0, 1, 3], [1, 2, 1])
    kv.release([0, 1, 3])
    assert np.all(kv.refs() == 0) and np.all(kv.lengths() == 0)
    with pytest.raises(ValueError):
        kv.fork([0], [1], [5], [0])
    with pytest.raises(RuntimeError):
        kv.fork([0, 1, 2, 3], [0] * 4, [0] * 4, [8 * page] * 4)
    with pytest.raises(ValueError):
        kv.append(0, C.ptr, [1, 1], [0, 1, 2], hq)
    with pytest.raises(ValueError):
        kv.extend([5], [1])
    with pytest.raises(ValueError):
        kv.attention(0, C.ptr, [0, 1], [0, 1], hq, S.ptr)
    kv.fork([], [], [], [])
    assert np.all(kv.refs() == 0) and kv.compact() == 0
    kv.close()


def test_cache_calls_from_stream_to_stream(hk_lib):
    """PagedKV's calls on alternating streams, each with other sequences: none overtakes the arguments or the
    workspace of the one before."""
    from runtime import hip, paged

    announce("paged cache: stream to stream")
    rng = np.random.default_rng(71)
    hq, hkv, dim, page = 4, 2, 64, 16
    kv = paged.PagedKV(layers=1, kv_heads=hkv, head_dim=dim, page_size=page, pages=400, seqs=6, table_width=70)
    lengths = [900, 20, 1000, 3, 700, 64]
    streams = []
    for _ in range(2):
        handle = ctypes.c_void_p()
        hip.check(hk_lib.hk_stream_create(ctypes.byref(handle)), "hk_stream_create")
        streams.append(handle.value)
    o = {"k": np.zeros((1, 400, hkv, page, dim)), "v": np.zeros((1, 400, hkv, page, dim)),
         "table": np.full((6, 70), -1, np.int32), "length": np.zeros(6, np.int32), "refs": np.zeros(400, np.int32)}
    first = np.cumsum([0] + lengths)
    x = _bits(rng.normal(size=(first[-1], hq + 2 * hkv, dim)))
    IN = _dev(x)
    row = 2 * (hq + 2 * hkv) * dim
    assert oracle.fork(o, range(6), range(6), [0] * 6, lengths) == (0, 0)
    kv.extend(range(6), lengths, streams[0])
    for s in range(6):  # a sequence a call, from stream to stream
        kv.append(0, IN.ptr + int(first[s]) * row, [s], [0, lengths[s]], hq, stream=streams[s % 2])
    oracle.append(o, 0, _floats(x), range(6), first, hq, None, None, lambda rows, which: rows)
    batches = [[s] for s in range(6)] + [[5, 0], [2, 4, 1], [3, 0, 2]]
    q = _bits(rng.normal(size=(len(batches), 3, hq, dim)))
    Q, OUT, SIZE = _dev(q), _dev(np.zeros(q.shape, np.uint16)), 2 * 3 * hq * dim
    for i, batch in enumerate(batches):
        kv.attention(0, Q.ptr + i * SIZE, batch, np.arange(len(batch) + 1), hq, OUT.ptr + i * SIZE, stream=streams[i % 2])
    for stream in streams:
        hip.check(hk_lib.hk_stream_sync(stream), "sync")
    got = _floats(OUT.read(np.uint16, q.size).reshape(q.shape))
    for i, batch in enumerate(batches):
        n = len(batch)
        want, _, spread = oracle.attention(o, 0, _floats(q[i, :n]), batch, np.arange(n + 1), dim**-0.5)
        # (a score's float32 error is below 64 2^-24 5^2 64 / 8 < 2^-10 for these draws)
        tol = 2.0**-8 * (np.abs(want) + spread) + (2.0**-9 + 2.0**-18) * spread + 1e-30
        assert np.all(np.abs(got[i, :n] - want) <= tol)
    kv.close()
    for stream in streams:
        hip.check(hk_lib.hk_stream_destroy(stream), "hk_stream_destroy")


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("why", ["full", "bad entry"])
def test_a_refused_fork_stops_the_steps_appends(hk_lib, why, captured):
    """A step enqueued in one go, and captured: after a fork that was refused the appends change neither the pages that
    two sequences share nor the queries' memory, and once there is room the same step goes through."""
    from runtime import hip, paged

    announce(f"paged cache: a refused fork, {why}, captured {captured}")
    rng = np.random.default_rng(81)
    hq, hkv, dim, page = 4, 2, 64, 16
    cache = Cache(rng, layers=2, pages=3, kv_heads=hkv, page=page, dim=dim, seqs=3, width=2, poison=False)
    # sequence 0 and 1: one full page that they share; 2: two pages.  Two more tokens need two pages more.
    cache.o["table"][:] = [[2, -1], [2, -1], [0, 1]]
    cache.o["refs"][:] = (1, 1, 2)
    cache.o["length"][:] = (16, 16, 20)
    for layer in (0, 1):
        cache.fill(rng, layer)
    cache.upload()
    x = _bits(rng.normal(size=(2, hq + 2 * hkv, dim)))
    IN, FIRST, STATUS = _dev(x), _dev(np.array([0, 1, 2], np.int32)), _dev(np.full(2, -9, np.int32))
    Q, GROW = _dev(np.full((2, hq, dim), 0x4242, np.uint16)), _dev(np.array([1, 1 if why == "full" else -1], np.int32))
    SEQ = _dev(np.array([0, 1], np.int32))
    cache.c.status = STATUS.ptr
    handle = ctypes.c_void_p()
    hip.check(hk_lib.hk_stream_create(ctypes.byref(handle)), "hk_stream_create")
    stream = handle.value
    lib, c, ws = paged.lib(), ctypes.byref(cache.c), cache.bufs["workspace"].ptr
    _sync()

    def enqueue():
        hip.check(lib.hk_paged_fork(c, SEQ.ptr, None, None, GROW.ptr, 2, STATUS.ptr, ws, stream), "hk_paged_fork")
        for layer in (0, 1):
            hip.check(lib.hk_paged_append(c, layer, IN.ptr, (hq + 2 * hkv) * dim, None, None, 0, SEQ.ptr, FIRST.ptr, 2, 2, hq,
                                          Q.ptr, hq * dim, stream), "hk_paged_append")

    graph = Graph(stream) if captured else None
    if captured:
        with graph:
            enqueue()

    def step():
        graph.replay() if captured else enqueue()
        hip.check(hk_lib.hk_stream_sync(stream), "sync")
        return tuple(STATUS.read(np.int32, 2).tolist())

    for _ in range(2):
        n = [int(v) for v in cache.o["length"][:2]]
        grow = [1, 1 if why == "full" else -1]
        want = oracle.fork(cache.o, [0, 1], [0, 1], n, grow)
        assert step() == want and want[0] == (paged.FULL if why == "full" else paged.BAD_ENTRY)
        same(cache)
        assert np.all(Q.read(np.uint16, 2 * hq * dim) == 0x4242)
    # room: sequence 2 is freed, and no count is below zero
    cache.c.status = None
    assert fork(cache, [2], [2], [0], [0]) == oracle.fork(cache.o, [2], [2], [0], [0]) == (0, 0)
    cache.c.status = STATUS.ptr
    GROW.write(np.array([1, 1], np.int32))
    assert step() == oracle.fork(cache.o, [0, 1], [0, 1], [16, 16], [1, 1]) == (0, 0)
    for layer in (0, 1):
        want = oracle.append(cache.o, layer, _floats(x), [0, 1], [0, 1, 2], hq, None, None, lambda rows, which: rows)
    same(cache)
    np.testing.assert_array_equal(Q.read(np.uint16, 2 * hq * dim).reshape(2, hq, dim), _bits(want))
    if captured:
        graph.close()
    hip.check(hk_lib.hk_stream_destroy(stream), "hk_stream_destroy")


def test_cache_calls_after_their_stream_is_gone(hk_lib):
    """PagedKV's calls, each on a stream of its own that is destroyed before the next one."""
    from runtime import hip, paged

    announce("paged cache: streams that are gone")
    rng = np.random.default_rng(91)
    hq, hkv, dim, page = 4, 2, 64, 16
    kv = paged.PagedKV(layers=1, kv_heads=hkv, head_dim=dim, page_size=page, pages=30, seqs=3, table_width=12)
    x = _bits(rng.normal(size=(90, hq + 2 * hkv, dim)))
    q = _bits(rng.normal(size=(3, hq, dim)))
    IN, Q, OUT = _dev(x), _dev(q), _dev(np.zeros(q.shape, np.uint16))

    def on_a_stream(call):
        handle = ctypes.c_void_p()
        hip.check(hk_lib.hk_stream_create(ctypes.byref(handle)), "hk_stream_create")
        call(handle.value)
        hip.check(hk_lib.hk_stream_sync(handle.value), "sync")
        hip.check(hk_lib.hk_stream_destroy(handle.value), "hk_stream_destroy")

    on_a_stream(lambda s: kv.extend([0, 1, 2], [60, 9, 21], s))
    on_a_stream(lambda s: kv.append(0, IN.ptr, [0, 1, 2], [0, 60, 69, 90], hq, stream=s))
    on_a_stream(lambda s: kv.attention(0, Q.ptr, [0, 1, 2], [0, 1, 2, 3], hq, OUT.ptr, stream=s))
    on_a_stream(kv.compact)
    assert kv.lengths().tolist() == [60, 9, 21]
    o = {"k": np.zeros((1, 30, hkv, page, dim)), "v": np.zeros((1, 30, hkv, page, dim)),
         "table": np.full((3, 12), -1, np.int32), "length": np.zeros(3, np.int32), "refs": np.zeros(30, np.int32)}
    assert oracle.fork(o, range(3), range(3), [0] * 3, [60, 9, 21]) == (0, 0)
    oracle.append(o, 0, _floats(x), range(3), [0, 60, 69, 90], hq, None, None, lambda rows, which: rows)
    got = _floats(OUT.read(np.uint16, q.size).reshape(q.shape))
    want, _, spread = oracle.attention(o, 0, _floats(q), range(3), range(4), dim**-0.5)
    # (a score's float32 error is below 64 2^-24 5^2 64 / 8 < 2^-10 for these draws)
    assert np.all(np.abs(got - want) <= 2.0**-8 * (np.abs(want) + spread) + (2.0**-9 + 2.0**-18) * spread + 1e-30)
    kv.close()
