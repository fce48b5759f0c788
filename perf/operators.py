"""Performance cases of the paged KV cache: its append, its attention, forking and compacting it.

``listed()`` names twelve calls, ``draw(rng)`` gives more of the same ranges.  ``prepare`` builds what a serving
program holds before the call (the page pools, tables, lengths and reference counts, the batch, the workspace), all of
it on the GPU and from the seed.  ``run`` is one call: with ``own`` false in plain float32 torch, with ``own`` true
through ``include/hk_paged.h``.  ``exact`` is the same result in float64, computed sequence by sequence.

The cache: sequence s has ``length[s]`` tokens, token j of it in slot ``j % page`` of page ``table[s, j // page]``; a
layer's pool is [pages, kv heads, page, head dim], bf16 or e4m3 with one scale per kv head, and ``refs[p]`` counts the
table entries that name page p.  Kinds of case:

- ``attention``  new tokens of a batch of sequences over their cached slots, causal, all sequences of their own lengths
- ``append``     new rows of the QKV projection: RoPE on queries and keys, keys and values into their pages
- ``fork``       sequences become prefixes of others, with pages for more tokens: full pages shared, partial ones copied
- ``compact``    the live pages move into the first ones of the pools, tables and counts follow
"""

import ctypes
import math
import random
import sys
from pathlib import Path

import torch

own = False

# bytes of device memory that the calls may use while they run, zero before the first (HK_PAGED_WORKSPACE)
WORKSPACE = 96 << 20

# (q heads, kv heads, head dim)
HEADS = {"14x2x64": (14, 2, 64), "9x3x64": (9, 3, 64), "32x8x64": (32, 8, 64), "32x8x128": (32, 8, 128),
         "28x4x128": (28, 4, 128), "16x16x128": (16, 16, 128)}


def listed():
    return [
        # the smallest call: one chat's next token, a short history, a small model
        {"name": "attention_token", "kind": "attention", "heads": "14x2x64", "page": 16, "e4m3": False, "seqs": 1,
         "new": 1, "length": 71, "window": 0},
        # a server's decode step: many chats of mixed ages
        {"name": "attention_decode_48", "kind": "attention", "heads": "32x8x128", "page": 64, "e4m3": False,
         "seqs": 48, "new": 1, "length": 9001, "window": 0},
        # the same with the cache in eight bits and more, shorter chats
        {"name": "attention_decode_e4m3_190", "kind": "attention", "heads": "28x4x128", "page": 32, "e4m3": True,
         "seqs": 190, "new": 1, "length": 4003, "window": 0},
        # a guess of five tokens per chat checked at once
        {"name": "attention_verify_16x5", "kind": "attention", "heads": "14x2x64", "page": 16, "e4m3": False,
         "seqs": 16, "new": 5, "length": 6011, "window": 0},
        # prompts in pieces beside chats in decode, a sliding window
        {"name": "attention_mixed_window", "kind": "attention", "heads": "32x8x64", "page": 32, "e4m3": False,
         "seqs": 9, "new": 701, "length": 5003, "window": 2047},
        # a piece of a very long prompt over what is cached of it
        {"name": "attention_prompt_2039", "kind": "attention", "heads": "32x8x128", "page": 128, "e4m3": False,
         "seqs": 1, "new": 2039, "length": 30011, "window": 0},
        # a decode step's new rows
        {"name": "append_token_61", "kind": "append", "heads": "14x2x64", "page": 16, "e4m3": False, "seqs": 61,
         "new": 1, "length": 37},
        # pieces of prompts into a cache in eight bits
        {"name": "append_chunks_e4m3", "kind": "append", "heads": "32x8x128", "page": 64, "e4m3": True, "seqs": 5,
         "new": 1907, "length": 2011},
        # a decode step's new pages: every sequence goes on by one token
        {"name": "fork_step_64", "kind": "fork", "heads": "14x2x64", "layers": 24, "page": 16, "seqs": 64, "from": 64,
         "grow": 1, "length": 611},
        # several answers to each of a few prompts: the prompts' pages shared, each answer its own last page
        {"name": "fork_answers_24x8", "kind": "fork", "heads": "32x8x128", "layers": 16, "page": 64, "seqs": 192,
         "from": 24, "grow": 2, "length": 903},
        # a small pool put in order
        {"name": "compact_512", "kind": "compact", "heads": "14x2x64", "layers": 24, "page": 16, "pages": 512,
         "live": 0.6},
        # a server's pool after its busy hour: half the pages free, to be given back
        {"name": "compact_1900", "kind": "compact", "heads": "32x8x128", "layers": 8, "page": 64, "pages": 1900,
         "live": 0.5},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "attention", "append", "append", "fork", "compact"))
    heads, page = rng.choice(sorted(HEADS)), rng.choice((16, 32, 64, 128))
    hq, hkv, d = HEADS[heads]
    case = {"kind": kind, "heads": heads, "page": page}
    if kind == "attention":
        new = rng.choice((1, 1, rng.randint(2, 8), _log_int(rng, 9, 2039)))
        length = new + _log_int(rng, 1, 9000 if new < 9 else 28000)
        most = min(190, (1 << 30) // (hq * new * length), (1 << 28) // (hkv * d * length))  # scores; cached values
        return dict(case, e4m3=rng.random() < 0.4, seqs=_log_int(rng, 1, max(1, most)), new=new, length=length,
                    window=rng.choice((0, 0, rng.randint(1, length))))
    if kind == "append":
        new = _log_int(rng, 1, 1907)
        return dict(case, e4m3=rng.random() < 0.5, seqs=_log_int(rng, 1, min(190, 9500 // new)), new=new,
                    length=new + _log_int(rng, 1, 300))
    layers = rng.choice((4, 8, 24)) if hkv * d < 512 else rng.choice((2, 8))
    if kind == "fork":
        seqs = _log_int(rng, 1, 192)
        step = rng.random() < 0.4
        return dict(case, layers=layers, seqs=seqs, **{"from": seqs if step else rng.randint(1, seqs)},
                    grow=rng.randint(1, 40), length=_log_int(rng, 2, 1000))
    most = min(16000, (1 << 30) // (layers * hkv * page * d))
    return dict(case, layers=layers, pages=_log_int(rng, 33, most), live=round(rng.uniform(0.1, 0.9), 3))


# ---- sizes that follow from a case ----


def _plan(case):
    """Lengths and new tokens of the batch's sequences: the last one is the longest, the others are younger, and in a
    batch of prompts' pieces every third sequence has a piece and the rest are in decode."""
    rng = random.Random("%s %s %s" % (case["seqs"], case["new"], case["length"]))
    n, most, new = case["seqs"], case["length"], case["new"]
    count = [new if new < 9 or i % 3 == (n - 1) % 3 else 1 for i in range(n)]
    count = [c if i == n - 1 or c == 1 else rng.randint(max(1, c // 2), c) for i, c in enumerate(count)]
    length = [max(c, _log_int(rng, max(1, most // 16), most)) for c in count]
    length[-1] = most
    return length, count


def _fork_plan(case):
    """The longest prefix is the whole of the first parent; the others vary."""
    rng = random.Random("%s %s %s" % (case["seqs"], case["from"], case["length"]))
    n, parents, most = case["seqs"], case["from"], case["length"]
    lengths = [most] + [rng.randint(max(1, most // 2), most) for _ in range(parents - 1)]
    if parents == n:  # the next step: every sequence goes on from itself
        return lengths, list(range(n)), list(range(n)), lengths
    parent = [i % parents for i in range(n)]
    return lengths, [parents + i for i in range(n)], parent, [lengths[p] for p in parent]


# ---- inputs ----


class _Draws:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32).mul_(std)

    def bf16(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.bfloat16).mul_(std)

    def scales(self, n):
        return (0.5 + torch.rand(n, generator=self.gen, device="cuda")) / 64.0

    def permutation(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda").to(torch.int32)

    def pool(self, shape, scale):
        """Normal keys or values of one layer, [pages, kv heads, page, head dim], as the cache holds them."""
        x = self.bf16(*shape)
        if scale is None:
            return x
        out = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn)
        for h in range(shape[1]):
            out[:, h] = (x[:, h].float() / scale[h]).clamp_(-448, 448).to(torch.float8_e4m3fn)
        return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(d, lengths, page, spare):
    """Pages of the sequences in a random order: (table, lengths, pages in the pool)."""
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + spare, max(need) + 2
    order = d.permutation(pages)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, _ints(lengths), pages


def _batch_state(case, seed):
    """A batch of sequences over one layer's pools."""
    d = _Draws(seed)
    hq, hkv, dim = HEADS[case["heads"]]
    length, count = _plan(case)
    table, lengths, pages = _tables(d, length, case["page"], 3)
    k_scale = v_scale = None
    if case["e4m3"]:
        k_scale, v_scale = d.scales(hkv), d.scales(hkv)
    shape = (pages, hkv, case["page"], dim)
    first = [0]
    for c in count:
        first.append(first[-1] + c)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[table[table >= 0].long()] = 1
    return d, dict(k=d.pool(shape, k_scale), v=d.pool(shape, v_scale), k_scale=k_scale, v_scale=v_scale, refs=refs,
                   table=table, length=lengths, first=_ints(first), seqs=_ints(range(len(length))), tokens=first[-1])


def _rope(slots, dim, dtype):
    inv = 1.0 / (10000.0 ** (torch.arange(dim // 2, device="cuda", dtype=torch.float64) / (dim // 2)))
    angle = torch.arange(slots, device="cuda", dtype=torch.float64)[:, None] * inv
    return angle.cos().to(dtype), angle.sin().to(dtype)


def _inputs(case, seed):
    hq, hkv, dim = HEADS[case["heads"]]
    page = case["page"]
    if case["kind"] in ("attention", "append"):
        d, state = _batch_state(case, seed)
        if case["kind"] == "attention":
            # queries that single out some of the keys, as trained heads' do: scores of standard deviation 2
            state["q"] = d.bf16(state["tokens"], hq, dim, std=2.0)
        else:
            state["qkv"] = d.bf16(state["tokens"], hq + 2 * hkv, dim)
        return state
    d = _Draws(seed)
    if case["kind"] == "fork":
        lengths, child, parent, keep = _fork_plan(case)
        grown = [-(-(k + case["grow"]) // page) for k in keep]
        table, length, pages = _tables(d, lengths, page, sum(grown) + 5)
        width = max(max(grown), table.shape[1])
        rows = max(child) + 1
        wide = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        wide[:table.shape[0], :table.shape[1]] = table
        length = torch.cat((length, torch.zeros(rows - len(lengths), dtype=torch.int32, device="cuda")))
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[table[table >= 0].long()] = 1
        state = dict(table=wide, length=length, refs=refs, child=_ints(child), parent=_ints(parent), keep=_ints(keep),
                     grow=_ints([case["grow"]] * len(child)))
    else:
        pages = case["pages"]
        live = max(1, int(case["live"] * pages))
        seqs = max(1, live // 24)
        width = -(-live // seqs)
        order = d.permutation(pages)[:live]
        table = torch.full((seqs * width,), -1, dtype=torch.int32, device="cuda")
        table[:live] = order
        table = table.view(seqs, width).contiguous()
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[order.long()] = 1
        # the first sequence has been forked: its row is there twice
        table = torch.cat((table, table[:1]))
        refs[table[0][table[0] >= 0].long()] += 1
        state = dict(table=table, refs=refs, length=(table >= 0).sum(1, dtype=torch.int32) * page)
    shape = (case["layers"], pages, hkv, page, dim)
    state.update(k=d.bf16(*shape), v=d.bf16(*shape))
    return state


def prepare(case, seed):
    hq, hkv, dim = HEADS[case["heads"]]
    state = dict(_inputs(case, seed), kind=case["kind"], hq=hq, hkv=hkv, dim=dim, page=case["page"])
    state["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    if case["kind"] == "attention":
        state.update(max_new=case["new"], slots=case["length"], window=case["window"], scale=dim ** -0.5,
                     out=torch.empty_like(state["q"]),
                     lse=torch.empty(state["q"].shape[:2], dtype=torch.float32, device="cuda"))
    elif case["kind"] == "append":
        cos, sin = _rope(state["table"].shape[1] * case["page"], dim, torch.float32)
        state.update(cos=cos, sin=sin, max_new=case["new"],
                     q=torch.empty(state["tokens"], hq, dim, dtype=torch.bfloat16, device="cuda"))
    elif case["kind"] == "fork":
        state["status"] = torch.empty(2, dtype=torch.int32, device="cuda")
    else:
        state.update(table_out=torch.empty_like(state["table"]), refs_out=torch.empty_like(state["refs"]),
                     live=torch.empty(1, dtype=torch.int32, device="cuda"))
    if own:
        state["cache"] = _describe(state)
    torch.cuda.synchronize()
    return state


# ---- the framework's calls ----


def _package():
    here = str(Path(__file__).resolve().parents[1] / "hawkpoint-npu-llm_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    from runtime import hip, paged

    return hip, paged


def _describe(s):
    """The cache as the calls take it: a description of the program's own memory."""
    hip, paged = _package()
    hip.init(0)
    k, scale = s["k"], s.get("k_scale")
    pages, page_stride = s["refs"].numel(), k[0].stride(0) if k.dim() == 5 else k.stride(0)
    return paged.PagedCache(
        k=k.data_ptr(), v=s["v"].data_ptr(), k_scale=None if scale is None else scale.data_ptr(),
        v_scale=None if scale is None else s["v_scale"].data_ptr(), table=s["table"].data_ptr(),
        length=s["length"].data_ptr(), refs=s["refs"].data_ptr(),
        layer_stride=k.stride(0) if k.dim() == 5 else pages * page_stride, page_stride=page_stride,
        layers=k.shape[0] if k.dim() == 5 else 1, kv_heads=s["hkv"], head_dim=s["dim"], page_size=s["page"],
        pages=pages, seqs=s["table"].shape[0], table_width=s["table"].shape[1],
        dtype=paged.BF16 if scale is None else paged.E4M3)


def _own(s):
    hip, paged = _package()
    lib, cache, kind = paged.lib(), ctypes.byref(s["cache"]), s["kind"]
    if kind == "attention":
        hip.check(lib.hk_paged_attention(
            cache, 0, s["q"].data_ptr(), s["hq"] * s["dim"], s["seqs"].data_ptr(), s["first"].data_ptr(),
            s["seqs"].numel(), s["tokens"], s["max_new"], s["hq"], s["scale"], s["window"], s["out"].data_ptr(),
            s["hq"] * s["dim"], s["lse"].data_ptr(), s["workspace"].data_ptr(), None), "hk_paged_attention")
        return {"out": s["out"], "lse": s["lse"]}
    if kind == "append":
        hip.check(lib.hk_paged_append(
            cache, 0, s["qkv"].data_ptr(), s["qkv"].stride(0), s["cos"].data_ptr(), s["sin"].data_ptr(),
            s["cos"].shape[0], s["seqs"].data_ptr(), s["first"].data_ptr(), s["seqs"].numel(), s["tokens"], s["hq"],
            s["q"].data_ptr(), s["q"].stride(0), None), "hk_paged_append")
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if kind == "fork":
        hip.check(lib.hk_paged_fork(
            cache, s["child"].data_ptr(), s["parent"].data_ptr(), s["keep"].data_ptr(), s["grow"].data_ptr(),
            s["child"].numel(), s["status"].data_ptr(), s["workspace"].data_ptr(), None), "hk_paged_fork")
        return _bits(s, s["table"], s["refs"], length=s["length"], status=s["status"])
    hip.check(lib.hk_paged_compact(
        cache, s["table_out"].data_ptr(), s["refs_out"].data_ptr(), s["live"].data_ptr(), s["workspace"].data_ptr(),
        None), "hk_paged_compact")
    return _bits(s, s["table_out"], s["refs_out"], live=s["live"])


def _bits(s, table, refs, **more):
    return dict(more, k=s["k"].view(torch.int16), v=s["v"].view(torch.int16), table=table, refs=refs)


# ---- the same in plain torch ----


def _plain_attention(s):
    hq, hkv, dim, page, n, new, slots = s["hq"], s["hkv"], s["dim"], s["page"], s["seqs"].numel(), s["max_new"], s["slots"]
    group, rows = hq // hkv, s["table"][s["seqs"].long()]
    length, first = s["length"][s["seqs"].long()].long(), s["first"].long()
    count = first[1:] - first[:-1]
    slot = torch.arange(slots, device="cuda")
    held = rows[:, slot // page].long()  # [n, slots]
    there = (held >= 0) & (slot < length[:, None])

    def cached(pool, scale):
        x = pool[held.clamp_min(0), :, slot % page].float()  # [n, slots, kv heads, dim]
        if scale is not None:
            x = x * scale[:, None]
        return torch.where(there[:, :, None, None], x, 0.0).transpose(1, 2)

    token = torch.arange(new, device="cuda")
    at = (first[:-1, None] + token).clamp_max(s["tokens"] - 1)  # [n, new] rows of q
    q = s["q"][at].float().view(n, new, hkv, group, dim).permute(0, 2, 1, 3, 4).reshape(n, hkv, new * group, dim)
    position = (length - count)[:, None] + token
    seen = there[:, None, :] & (slot <= position[:, :, None])
    if s["window"]:
        seen = seen & (slot > position[:, :, None] - s["window"])
    seen = seen[:, None, :, None, :]
    score = torch.matmul(q, cached(s["k"], s["k_scale"]).transpose(2, 3)).view(n, hkv, new, group, slots)
    score.mul_(s["scale"]).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, hkv, new * group, slots), cached(s["v"], s["v_scale"])).view(n, hkv, new, group, dim)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + total.log())[..., 0]  # a row that sees nothing: log 0
    has = token < count[:, None]
    s["out"][at[has]] = out.permute(0, 2, 1, 3, 4).reshape(n, new, hq, dim)[has].to(torch.bfloat16)
    s["lse"][at[has]] = lse.permute(0, 2, 1, 3).reshape(n, new, hq)[has]
    return {"out": s["out"], "lse": s["lse"]}


def _places(s):
    """Position, page and slot of each new token."""
    first, seqs = s["first"].long(), s["seqs"].long()
    token = torch.arange(s["tokens"], device="cuda")
    entry = torch.searchsorted(first[1:].contiguous(), token, right=True)
    position = s["length"].long()[seqs[entry]] - first[entry + 1] + token
    return position, s["table"][seqs[entry], position // s["page"]].long(), position % s["page"]


def _plain_append(s):
    hq, hkv, dim = s["hq"], s["hkv"], s["dim"]
    position, page, slot = _places(s)
    x = s["qkv"].float()
    cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]
    a, b = x[:, :hq + hkv, :dim // 2], x[:, :hq + hkv, dim // 2:]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    s["q"].copy_(turned[:, :hq])

    def store(pool, rows, scale):
        if scale is None:
            pool[page, :, slot] = rows.to(torch.bfloat16)
        else:  # (indexed stores of bytes: torch has none of float8)
            rows = (rows / scale[:, None]).clamp_(-448, 448).to(torch.float8_e4m3fn)
            pool.view(torch.uint8)[page, :, slot] = rows.view(torch.uint8)

    store(s["k"], turned[:, hq:], s["k_scale"])
    store(s["v"], x[:, hq + hkv:], s["v_scale"])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _count(ids, size):
    return torch.bincount(ids.reshape(-1), minlength=size).to(torch.int32)


def _plain_fork(s):
    page, table, n = s["page"], s["table"], s["child"].numel()
    pages, width = s["refs"].numel(), table.shape[1]
    child, parent, keep, grow = (s[x].long() for x in ("child", "parent", "keep", "grow"))
    column = torch.arange(width, device="cuda")
    full, total = (keep // page)[:, None], ((keep + grow + page - 1) // page)[:, None]
    part, source, before = keep % page > 0, table[parent].long(), table[child].long()
    shared = column < full
    refs = s["refs"] - _count(before[before >= 0], pages) + _count(source[shared], pages)
    # a partial page that nobody else keeps goes to the first that wants it; the others copy it
    index = torch.arange(n, device="cuda")
    wanted = torch.where(part, source.gather(1, full.clamp_max(width - 1))[:, 0], pages)
    first = torch.full((pages + 1,), n, device="cuda").scatter_reduce_(0, wanted, index, "amin")
    padded = torch.cat((refs, refs.new_ones(1)))
    taken = part & (padded[wanted] == 0) & (first[wanted] == index)
    here = (column == full) & taken[:, None]
    refs = refs + _count(source[here], pages)
    fresh = (column >= full) & (column < total) & ~here
    free = (refs > 0).sort(stable=True).indices
    order = torch.cumsum(fresh.reshape(-1), 0).view(n, width) - 1
    new = torch.where(fresh, free[order.clamp(0, pages - 1)], torch.where(shared | here, source, -1))
    s["refs"].copy_(refs + _count(new[fresh], pages))
    copies = (part & ~taken).nonzero()[:, 0]
    src, dst = wanted[copies], new[copies, keep[copies] // page]
    slot = (torch.arange(page, device="cuda") < (keep % page)[copies, None])[None, :, None, :, None]
    for_all = ("k", "v")
    s.update({x: _copied(s[x], src, dst, slot) for x in for_all})
    table[child] = new.to(torch.int32)
    s["length"][child] = (keep + grow).to(torch.int32)
    s["status"].zero_()
    return _bits(s, table, s["refs"], length=s["length"], status=s["status"])


def _copied(pool, src, dst, slot):
    pool[:, dst] = torch.where(slot, pool[:, src], pool[:, dst])
    return pool


def _plain_compact(s):
    live = s["refs"] > 0
    total = live.sum()
    ids = torch.arange(live.numel(), device="cuda")
    holes, movers = ((ids < total) & ~live).nonzero()[:, 0], ((ids >= total) & live).nonzero()[:, 0]
    place = ids.clone()
    place[movers] = holes
    named = (s["table"] >= 0)
    s["table_out"].copy_(torch.where(named, place[s["table"].clamp_min(0).long()], s["table"].long()))
    s["refs_out"].zero_()
    s["refs_out"][place[live]] = s["refs"][live]
    s["live"].copy_(total.view(1))
    s["k"][:, holes] = s["k"][:, movers]
    s["v"][:, holes] = s["v"][:, movers]
    return _bits(s, s["table_out"], s["refs_out"], live=s["live"])


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "append": _plain_append, "fork": _plain_fork,
            "compact": _plain_compact}[state["kind"]](state)


# ---- what a call cannot do without ----


def _seen(case):
    """(slots read, (row, slot) pairs) of an attention case, of one head."""
    slots = pairs = 0
    window = case["window"]
    for length, count in zip(*_plan(case)):
        start = length - count
        low = max(0, start - window + 1) if window else 0
        slots += length - low
        if not window:
            pairs += count * start + count * (count + 1) // 2
        else:
            pairs += sum(min(window, start + i + 1) for i in range(count))
    return slots, pairs


def work(case):
    hq, hkv, dim = HEADS[case["heads"]]
    page, size = case["page"], 1 if case.get("e4m3") else 2
    if case["kind"] == "attention":
        slots, pairs = _seen(case)
        tokens = sum(_plan(case)[1])
        return {"bytes": 2 * size * hkv * dim * slots + 4 * tokens * hq * dim + 4 * tokens * hq + 4 * slots // page,
                "flops": 4 * hq * dim * pairs}
    if case["kind"] == "append":
        tokens = sum(_plan(case)[1])
        return {"bytes": tokens * dim * (2 * (hq + 2 * hkv) + 2 * hq + 2 * size * hkv) + 4 * tokens * dim,
                "flops": 3 * tokens * (hq + hkv) * dim}
    row = 2 * case["layers"] * hkv * dim * 2  # bytes of one slot, keys and values of all layers
    if case["kind"] == "fork":
        lengths, child, parent, keep = _fork_plan(case)
        entries = sum(-(-(k + case["grow"]) // page) for k in keep)
        # a sequence that goes on from itself keeps its last page, the others copy its slots
        copied = sum(k % page for c, p, k in zip(child, parent, keep) if c != p)
        return {"bytes": 2 * row * copied + 8 * entries + 8 * entries + 16 * len(keep), "flops": 0}
    live = max(1, int(case["live"] * case["pages"]))
    # of `live` pages anywhere in the pool, this many lie past the first `live` on average
    moved = live * (case["pages"] - live) / case["pages"]
    return {"bytes": 2 * row * page * moved + 8 * live + 8 * case["pages"], "flops": 0}


# ---- the same results in float64 ----


def _rows64(s, pool, scale, seq, n):
    """The first n slots of a sequence, [kv heads, n, dim]."""
    pages = s["table"][seq, :-(-n // s["page"])].long()
    x = pool[pages].double()  # [pages, kv heads, page, dim]
    if scale is not None:
        x = x * scale.double()[:, None, None]
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n]


def exact(case, seed):
    hq, hkv, dim = HEADS[case["heads"]]
    if case["kind"] not in ("attention", "append"):
        return None  # whole numbers and moved values: nothing is computed
    s = dict(_inputs(case, seed), page=case["page"])
    lengths, counts = _plan(case)
    group, row = hq // hkv, 0
    if case["kind"] == "attention":
        out = torch.zeros(s["tokens"], hq, dim, dtype=torch.float64, device="cuda")
        lse = torch.zeros(s["tokens"], hq, dtype=torch.float64, device="cuda")
        for i, (length, count) in enumerate(zip(lengths, counts)):
            low = 0 if not case["window"] else max(0, length - count - case["window"] + 1)
            k = _rows64(s, s["k"], s["k_scale"], i, length)[:, low:]
            v = _rows64(s, s["v"], s["v_scale"], i, length)[:, low:]
            ahead = torch.arange(low, length, device="cuda") - torch.arange(length - count, length, device="cuda")[:, None]
            hidden = ahead > 0
            if case["window"]:
                hidden |= ahead <= -case["window"]
            for h in range(hq):
                score = s["q"][row:row + count, h].double() @ k[h // group].T * dim ** -0.5
                score.masked_fill_(hidden, -math.inf)
                lse[row:row + count, h] = torch.logsumexp(score, 1)
                out[row:row + count, h] = torch.softmax(score, 1) @ v[h // group]
            row += count
        return {"out": out, "lse": lse}
    cos, sin = _rope(s["table"].shape[1] * s["page"], dim, torch.float64)
    q = torch.zeros(s["tokens"], hq, dim, dtype=torch.float64, device="cuda")
    k, v = s["k"].double(), s["v"].double()
    for i, (length, count) in enumerate(zip(lengths, counts)):
        at = torch.arange(length - count, length, device="cuda")
        x = torch.complex(*s["qkv"][row:row + count, :hq + hkv].double().chunk(2, -1))
        x = x * torch.complex(cos[at], sin[at])[:, None]
        x = torch.cat((x.real, x.imag), -1)
        q[row:row + count] = x[:, :hq]
        pages, slots = s["table"][i, at // s["page"]].long(), at % s["page"]
        for pool, new, scale in ((k, x[:, hq:], s["k_scale"]), (v, s["qkv"][row:row + count, hq + hkv:], s["v_scale"])):
            new = new.double()
            pool[pages, :, slots] = new if scale is None else (new / scale.double()[:, None]).clamp(-448, 448)
        row += count
    return {"q": q, "k": k, "v": v}
