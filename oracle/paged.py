"""The paged KV cache's operators in NumPy float64, slot by slot from their definitions (include/hk_paged.h).  This
build's own definition: the reference keeps one sequence's cache and has no counterpart.

A cache is a dict: ``k`` and ``v`` [layers, pages, kv heads, page, dim] as float values, ``table`` [seqs, width],
``length`` [seqs], ``refs`` [pages] int32."""

import numpy as np

__all__ = ["append", "attention", "compact", "fork", "e4m3", "from_e4m3"]


def from_e4m3(codes):
    """OCP e4m3 bytes as float64: 4 exponent bits (bias 7), 3 mantissa bits, no infinity, 0x7f and 0xff NaN."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    x = np.where(e == 0, m * 2.0**-9, (8 + m) * 2.0 ** (e - 10.0))
    x = np.where((c & 0x7F) == 0x7F, np.nan, x)
    return np.where(c & 0x80, -x, x)


_E4M3 = from_e4m3(np.arange(127))  # 0 .. 448, ascending


def e4m3(x):
    """The nearest e4m3 byte (ties to even, saturated) of each value; NaN as 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.where(np.isnan(x), 0, x)), 448.0)
    hi = np.clip(np.searchsorted(_E4M3, a), 1, 126)
    lo = hi - 1
    down, up = a - _E4M3[lo], _E4M3[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(x), 0x7F, code | np.where(np.signbit(x), 0x80, 0))
    return code.astype(np.uint8)


def rows_of(first, b, tokens):
    f0 = min(max(int(first[b]), 0), tokens)
    return f0, min(max(int(first[b + 1]), f0), tokens)


def slots_of(cache, seq, upto):
    """(slot numbers, pages, slots in them) of the sequence's slots below ``upto`` whose page exists."""
    page = cache["k"].shape[3]
    j = np.arange(upto)
    held = cache["table"][seq, j // page] if upto else np.zeros(0, np.int32)
    ok = (held >= 0) & (held < cache["k"].shape[1])
    return j[ok], held[ok], j[ok] % page


def length_of(cache, seq):
    if not 0 <= seq < len(cache["length"]):
        return 0
    return min(max(int(cache["length"][seq]), 0), cache["table"].shape[1] * cache["k"].shape[3])


def attention(cache, layer, q, seqs, first, scale, window=0):
    """q [tokens, heads, dim] -> (out, lse, spread); spread [tokens, heads, dim] = sum_j p_j |v_j|, which scales the
    rounding of the probabilities.  Rows of no entry: spread -1, the others NaN."""
    tokens, heads, dim = q.shape
    kv_heads = cache["k"].shape[2]
    out, spread = np.full(q.shape, np.nan), np.full(q.shape, -1.0)
    lse = np.full((tokens, heads), np.nan)
    for b, seq in enumerate(seqs):
        f0, f1 = rows_of(first, b, tokens)
        length = length_of(cache, seq)
        slot, page, at = slots_of(cache, seq, length)
        for t in range(f0, f1):
            p = length - f1 + t
            see = slot <= p
            if window:
                see &= slot > p - window
            for h in range(heads):
                g = h // (heads // kv_heads)
                k, v = cache["k"][layer, page[see], g, at[see]], cache["v"][layer, page[see], g, at[see]]
                if not len(k):
                    out[t, h], spread[t, h], lse[t, h] = 0, 0, -np.inf
                    continue
                s = (k @ q[t, h]) * scale
                e = np.exp(s - s.max())
                out[t, h] = e @ v / e.sum()
                spread[t, h] = e @ np.abs(v) / e.sum()
                lse[t, h] = s.max() + np.log(e.sum())
    return out, lse, spread


def turn(x, cos, sin):
    a, b = np.split(x, 2, axis=-1)
    return np.concatenate((a * cos - b * sin, b * cos + a * sin), -1)


def append(cache, layer, qkv, seqs, first, q_heads, cos, sin, store):
    """qkv [tokens, q + 2 kv heads, dim]: turned queries (NaN where there are none); ``store`` turns key or value rows
    [kv heads, dim] and "k" / "v" into what the pools hold of them."""
    tokens = qkv.shape[0]
    kv_heads, page = cache["k"].shape[2], cache["k"].shape[3]
    out = np.full((tokens, q_heads, qkv.shape[2]), np.nan)
    for b, seq in enumerate(seqs):
        f0, f1 = rows_of(first, b, tokens)
        length = length_of(cache, seq)
        for t in range(f0, f1):
            p = length - f1 + t
            if p < 0:
                continue
            x = qkv[t].astype(np.float64)
            qk = x[:q_heads + kv_heads]
            if cos is not None:
                qk = turn(qk, cos[p].astype(np.float64), sin[p].astype(np.float64))
            out[t] = qk[:q_heads]
            held = cache["table"][seq, p // page]
            if 0 <= held < cache["k"].shape[1]:
                cache["k"][layer, held, :, p % page] = store(qk[q_heads:], "k")
                cache["v"][layer, held, :, p % page] = store(x[q_heads + kv_heads:], "v")
    return out


def fork(cache, child, parent, keep, grow):
    """(code, word) as hk_paged_fork's status; the cache is changed in place only for code 0."""
    table, length, refs = (cache[x].copy() for x in ("table", "length", "refs"))
    page, pages, seqs, width = cache["k"].shape[3], cache["k"].shape[1], len(length), table.shape[1]
    seen = set()
    for i, (c, q, k, g) in enumerate(zip(child, parent, keep, grow)):
        ok = 0 <= c < seqs and c not in seen and k >= 0 and g >= 0 and k + g <= width * page
        ok = ok and (k == 0 or (0 <= q < seqs and k <= length_of(cache, q)))
        if ok and k % page:
            ok = 0 <= cache["table"][q, k // page] < pages
        if not ok:
            return 1, i
        seen.add(c)
    is_page = lambda p: 0 <= p < pages  # noqa: E731
    for c in child:
        for p in cache["table"][c, :-(-length_of(cache, c) // page)]:
            if is_page(p):
                refs[p] -= 1
        table[c] = -1
    for c, q, k in zip(child, parent, keep):
        for j in range(k // page):
            table[c, j] = cache["table"][q, j]
            if is_page(table[c, j]):
                refs[table[c, j]] += 1
    kept = refs > 0
    copies, needed = [], []
    for c, q, k, g in zip(child, parent, keep, grow):
        at = k // page
        if k % page:
            p = cache["table"][q, at]
            if not kept[p] and refs[p] == 0:
                table[c, at], refs[p] = p, 1
                at += 1
            else:
                copies.append((p, c, at, k % page))
        needed += [(c, j) for j in range(at, -(-(k + g) // page))]
    free = np.flatnonzero(refs <= 0)
    if len(free) < len(needed):
        return 2, len(needed) - len(free)
    for (c, j), p in zip(needed, free):
        table[c, j], refs[p] = p, 1
    for p, c, j, n in copies:
        for pool in (cache["k"], cache["v"]):
            pool[:, table[c, j], :, :n] = pool[:, p, :, :n]
    for c, k, g in zip(child, keep, grow):
        length[c] = k + g
    cache.update(table=table, length=length, refs=refs)
    return 0, 0


def compact(cache):
    """Moves the live pages to the front in place; returns their number."""
    refs = cache["refs"]
    live = int((refs > 0).sum())
    place = np.arange(len(refs))
    place[np.flatnonzero(refs[live:] > 0) + live] = np.flatnonzero(refs[:live] <= 0)
    for pool in (cache["k"], cache["v"]):
        for p in np.flatnonzero(refs[live:] > 0) + live:
            pool[:, place[p]] = pool[:, p]
    new = np.zeros_like(refs)
    for p in np.flatnonzero(refs > 0):
        new[place[p]] = refs[p]
    t = cache["table"]
    named = (t >= 0) & (t < len(refs))
    cache["table"] = np.where(named, place[np.where(named, t, 0)], t).astype(np.int32)
    cache["refs"] = new
    return live
