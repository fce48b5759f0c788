"""ctypes binding of include/hk_paged.h: a paged KV cache, its append, its
attention, forking and compaction.

``lib()`` gives the calls on device pointers.  ``PagedKV`` owns one cache's
memory (pools, tables, lengths, counts, workspace) and makes the calls with
host arrays of sequence numbers and lengths; activations stay on the device.
The reference has no counterpart: its engine keeps one sequence's cache
(npu_llm/runtime/qwen_engine.py:52-63).
"""

import ctypes

import numpy as np

from runtime import hip

__all__ = ["EXPORTED", "BF16", "E4M3", "WORKSPACE", "DONE", "BAD_ENTRY", "FULL", "PagedCache", "PagedKV", "lib"]

BF16 = 0
E4M3 = 1
WORKSPACE = 100663296  # HK_PAGED_WORKSPACE
DONE, BAD_ENTRY, FULL = 0, 1, 2  # status words of hk_paged_fork

_vp = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64


class PagedCache(ctypes.Structure):
    _fields_ = [
        ("k", _vp),
        ("v", _vp),
        ("k_scale", _vp),
        ("v_scale", _vp),
        ("table", _vp),
        ("length", _vp),
        ("refs", _vp),
        ("layer_stride", _i64),
        ("page_stride", _i64),
        ("layers", _i32),
        ("kv_heads", _i32),
        ("head_dim", _i32),
        ("page_size", _i32),
        ("pages", _i32),
        ("seqs", _i32),
        ("table_width", _i32),
        ("dtype", _i32),
        ("status", _vp),
    ]


_SIGNATURES = {
    "hk_paged_append": (
        ctypes.c_int,
        [_vp, _i32, _vp, _i64, _vp, _vp, _i32, _vp, _vp, _i32, _i32, _i32, _vp, _i64, _vp],
    ),
    "hk_paged_attention": (
        ctypes.c_int,
        [_vp, _i32, _vp, _i64, _vp, _vp, _i32, _i32, _i32, _i32, ctypes.c_float, _i32, _vp, _i64, _vp, _vp, _vp],
    ),
    "hk_paged_fork": (ctypes.c_int, [_vp, _vp, _vp, _vp, _vp, _i32, _vp, _vp, _vp]),
    "hk_paged_compact": (ctypes.c_int, [_vp, _vp, _vp, _vp, _vp, _vp]),
}

EXPORTED = tuple(_SIGNATURES)

_bound = None


def lib():
    global _bound
    if _bound is None:
        handle = hip.lib()
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _bound = handle
    return _bound


def _i32s(values, n, name):
    a = np.asarray(values)
    if a.shape != (n,) or a.dtype.kind not in "iu":
        raise ValueError(f"{name} must be {n} whole numbers")
    if n and (a.min() < -(2**31) or a.max() >= 2**31):
        raise ValueError(f"{name} outside 32 bits")
    return np.ascontiguousarray(a, dtype=np.int32)


class PagedKV:
    """One paged cache: ``pages`` pages of ``page_size`` slots for every layer, shared by up to ``seqs`` sequences of
    at most ``table_width`` pages.  All sequences are empty at first.

    ``fork`` (and ``extend``, ``release`` in its terms) changes which pages the sequences hold, ``append`` stores new
    rows of the QKV projection, ``attention`` reads them, ``compact`` moves the live pages to the front.  Activations
    are device buffers of bf16 rows; ``first`` is the list of the entries' first rows, one longer than ``seqs``.

    A call waits for the one before (whatever its stream, which may be gone by then) before it hands its host arrays
    over: for one thread, and not for capture into a graph.  A program that counts microseconds keeps its arrays on the
    device and makes the calls of ``lib()``: here each layer's append and attention waits and copies them again.
    """

    def __init__(self, *, layers, kv_heads, head_dim, page_size, pages, seqs, table_width, dtype=BF16, k_scale=None,
                 v_scale=None, device=0):
        hip.init(device)
        self._lib = lib()
        if min(layers, kv_heads, head_dim, page_size, pages, seqs, table_width) <= 0:
            raise ValueError("cache sizes must be positive")
        if dtype not in (BF16, E4M3):
            raise ValueError("unknown dtype")
        if (dtype == E4M3) != (k_scale is not None) or (dtype == E4M3) != (v_scale is not None):
            raise ValueError("an e4m3 cache needs k_scale and v_scale, a bf16 cache takes none")
        page = kv_heads * page_size * head_dim
        size = layers * pages * page * (2 if dtype == BF16 else 1)
        self.bufs = {"k": hip.DeviceBuffer(size), "v": hip.DeviceBuffer(size), "length": hip.DeviceBuffer(4 * seqs),
                     "table": hip.DeviceBuffer(4 * seqs * table_width), "refs": hip.DeviceBuffer(4 * pages),
                     "workspace": hip.DeviceBuffer(WORKSPACE), "args": hip.DeviceBuffer(16 * (seqs + 1) + 64)}
        for name in ("length", "refs", "workspace"):
            self.bufs[name].zero()
        hip.check(self._lib.hk_memset(self.bufs["table"].ptr, 255, self.bufs["table"].nbytes), "hk_memset")
        for name, scale in (("k_scale", k_scale), ("v_scale", v_scale)):
            if scale is None:
                continue
            scale = np.ascontiguousarray(scale, dtype=np.float32)
            if scale.shape != (layers, kv_heads) or not np.all(np.isfinite(scale) & (scale > 0)):
                raise ValueError(f"{name} must be [layers, kv_heads], finite and positive")
            self.bufs[name] = hip.DeviceBuffer.from_array(scale)
        hip.check(self._lib.hk_stream_sync(None), "sync")  # (the calls may go to other streams)
        self._start, self._done = hip.Event(), hip.Event()  # _done: the end of the call before, on its stream
        self._start.record(None)
        self._done.record(None)
        ptr = {name: b.ptr for name, b in self.bufs.items() if name not in ("workspace", "args")}
        self.cache = PagedCache(layer_stride=pages * page, page_stride=page, layers=layers, kv_heads=kv_heads,
                                head_dim=head_dim, page_size=page_size, pages=pages, seqs=seqs,
                                table_width=table_width, dtype=dtype, **ptr)

    def _wait(self):
        """For the end of the call before.  By its event: its stream is the caller's, who may have destroyed it."""
        self._start.elapsed_ms(self._done)

    def _call(self, name, *args):
        """The last argument is the stream."""
        rc = getattr(self._lib, name)(ctypes.byref(self.cache), *args)
        self._done.record(args[-1])
        hip.check(rc, name)

    def _args(self, *arrays):
        """Device copies of a call's host arrays (None stays None), one behind the other, once the call before has read
        its own and is through with the workspace."""
        self._wait()
        given = [a for a in arrays if a is not None]
        if sum(a.nbytes for a in given) > self.bufs["args"].nbytes:
            raise ValueError("more entries than the cache has sequences")
        ptrs, at = [], 0
        for a in arrays:
            ptrs.append(None if a is None else self.bufs["args"].ptr + at)
            at += 0 if a is None else a.nbytes
        if given:
            self.bufs["args"].write(np.concatenate(given))
        return ptrs

    def fork(self, child, parent, keep, grow, stream=None):
        """Each child sequence becomes the first ``keep`` tokens of its parent with room for ``grow`` more, all at
        once; waits for the outcome.  ValueError for an entry that is not valid, RuntimeError when the pages do not
        suffice; nothing is changed then, and the rows that were to come have no place: an append of them would store
        over the last tokens there are."""
        n = len(child)
        if n == 0:
            return
        arrays = [_i32s(a, n, name) for a, name in ((child, "child"), (parent, "parent"), (keep, "keep"),
                                                    (grow, "grow"))]
        args = self._args(*arrays)
        status = self.bufs["args"].nbytes - 8
        self._call("hk_paged_fork", *args, n, self.bufs["args"].ptr + status, self.bufs["workspace"].ptr, stream)
        self._wait()
        code, what = self.bufs["args"].read(np.int32, 2, status)
        if code == BAD_ENTRY:
            raise ValueError(f"fork: entry {what} is not valid")
        if code == FULL:
            raise RuntimeError(f"fork: {what} pages are missing")

    def extend(self, seqs, counts, stream=None):
        """Room for ``counts`` new tokens of each sequence: the next step's."""
        length = self.lengths(stream)
        seqs = _i32s(seqs, len(seqs), "seqs")
        if len(seqs) and (seqs.min() < 0 or seqs.max() >= len(length)):
            raise ValueError("sequence outside the cache")
        self.fork(seqs, seqs, length[seqs], counts, stream)

    def release(self, seqs, stream=None):
        """Empties the sequences; pages that nobody else holds are free."""
        zero = np.zeros(len(seqs), np.int32)
        self.fork(seqs, seqs, zero, zero, stream)

    def append(self, layer, qkv, seqs, first, q_heads, *, rope=None, q_out=None, stream=None):
        """Stores the rows of ``qkv`` (device pointer, rows of q, k and v heads) as the last tokens of ``seqs``;
        ``rope``: (cos, sin, positions) device tables, ``q_out`` (device pointer) receives the turned queries."""
        n, c = len(seqs), self.cache
        first = _i32s(first, n + 1, "first")
        seqs = _i32s(seqs, n, "seqs")
        if len(np.unique(seqs)) < n:
            raise ValueError("a sequence is listed twice")
        args = self._args(seqs, first)
        cos, sin, positions = rope or (None, None, 0)
        width = (q_heads + 2 * c.kv_heads) * c.head_dim
        self._call("hk_paged_append", layer, qkv, width, cos, sin, positions, *args, n, int(first[-1]), q_heads, q_out,
                   q_heads * c.head_dim, stream)

    def attention(self, layer, q, seqs, first, q_heads, out, *, scale=None, window=0, lse=None, stream=None):
        """Attention of the rows of ``q`` (device pointer), the last tokens of ``seqs``, into ``out``."""
        n, c = len(seqs), self.cache
        first = _i32s(first, n + 1, "first")
        args = self._args(_i32s(seqs, n, "seqs"), first)
        width = q_heads * c.head_dim
        self._call("hk_paged_attention", layer, q, width, *args, n, int(first[-1]),
                   max(1, int(np.diff(first).max(initial=1))), q_heads, c.head_dim ** -0.5 if scale is None else scale,
                   window, out, width, lse, self.bufs["workspace"].ptr, stream)

    def compact(self, stream=None):
        """Moves the live pages to the front of the pool, in place; returns their number."""
        self._wait()
        live = self.bufs["args"].ptr + self.bufs["args"].nbytes - 8
        self._call("hk_paged_compact", self.cache.table, self.cache.refs, live, self.bufs["workspace"].ptr, stream)
        self._wait()
        return int(self.bufs["args"].read(np.int32, 1, self.bufs["args"].nbytes - 8)[0])

    def _read(self, name, stream):
        self._wait()
        hip.check(self._lib.hk_stream_sync(stream), "sync")  # (the caller may have made calls of lib() there)
        return self.bufs[name].read(np.int32, self.bufs[name].nbytes // 4)

    def lengths(self, stream=None):
        return self._read("length", stream)

    def refs(self, stream=None):
        return self._read("refs", stream)

    def table(self, stream=None):
        return self._read("table", stream).reshape(self.cache.seqs, self.cache.table_width)

    def close(self):
        for b in getattr(self, "bufs", {}).values():
            b.free()
        self.bufs = {}

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
