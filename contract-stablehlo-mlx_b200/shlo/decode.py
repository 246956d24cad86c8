"""The decoder operators: rotary positions, the paged key/value cache in 8 bits and
the attention that reads it, for hosts that generate token by token.

The *_noalloc functions take device tensors of the caller's own -- objects with
data_ptr(), shape, stride(), dtype, is_cuda, numel(), element_size() and is_contiguous(), as
a torch.Tensor has them; nothing here imports torch -- and queue their work on `stream` (a cudaStream_t as
an integer; 0 is the default stream) of the device that is current in CUDA. A tensor of another device is refused,
as far as it says where it lies (get_device()). They allocate nothing. Every one is one call
of include/shlo_cuda.h, whose comments say what it computes; errors raise ShloError.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import mlx as M
from . import run as Run
from ._lib import KvBatch, KvPool, ShloError, check, load

SCALINGS = {"none": 0, "linear": 1, "base": 2, "ramp": 3, "blend": 4}

_NAMES = {"torch.float16": M.dtF16, "torch.float32": M.dtF32, "torch.int32": M.dtI32, "torch.int64": M.dtI64,
          "torch.int8": M.dtI8}
_F16, _F32, _I8, _I32, _I64 = M.dtF16, M.dtF32, M.dtI8, M.dtI32, M.dtI64
_codes: dict = {}  # a dtype object seen before -> its code (None: not carried)


def _elsewhere(x, at):
    """x does not lie on device `at`, or does not say."""
    if not x.is_cuda:
        raise ShloError("a tensor in host memory: the decoder operators take device memory")
    if at is not None and hasattr(x, "get_device"):
        raise ShloError("a tensor on device %d, but device %d is the current one or the other tensors'" % (x.get_device(), at))


def _code(x, at):
    try:
        if x.get_device() != at:
            _elsewhere(x, at)
    except AttributeError:
        _elsewhere(x, at)
    d = x.dtype
    try:
        return _codes[d]
    except KeyError:
        return _codes.setdefault(d, _NAMES.get(str(d)))


def rope_phases(rot: int, base: float = 10000.0, scaling: str = "none", by: float = 1.0, trained: float = 0.0,
                fast: float = 32.0, slow: float = 1.0):
    """(phases int64 [rot / 2] on the host, factor): the plan of the rotary positions of a model."""
    if scaling not in SCALINGS:
        raise ShloError("rope phases: scaling %r not carried" % (scaling,))
    out = np.zeros(max(rot // 2, 1), np.int64)
    f = ctypes.c_float()
    check(load().shlo_rope_phases(rot, base, SCALINGS[scaling], by, trained, fast, slow,
                                  out.ctypes.data_as(ctypes.c_void_p), ctypes.byref(f)))
    return out, f.value


def _rows(x, what, at):
    """A float [tokens, heads, dim] whose last axis is contiguous: (shape, strides, type code)."""
    c, n, s = _code(x, at), x.shape, x.stride()
    if c != _F16 and c != _F32:
        raise ShloError("%s: %s not carried (float16 or float32)" % (what, x.dtype))
    if len(n) != 3:
        raise ShloError("%s: rank %d, [tokens, heads, dim] expected" % (what, len(n)))
    if s[2] != 1 and n[2] > 1:
        raise ShloError("%s: the last axis is strided" % what)
    return n, s, c


def _list(x, code, what, at):
    """A contiguous vector of a type: its length."""
    n = x.shape
    if _code(x, at) != code or len(n) != 1:
        raise ShloError("%s: %s of rank %d, a vector of int%d expected" % (what, x.dtype, len(n), 32 if code == M.dtI32 else 64))
    if n[0] > 1 and x.stride()[0] != 1:
        raise ShloError("%s: the last axis is strided" % what)
    return n[0]


def _tables(x, what, at):
    """int32 [sequences, pages], rows at any distance: (shape, row stride)."""
    n, s = x.shape, x.stride()
    if _code(x, at) != _I32 or len(n) != 2:
        raise ShloError("%s: %s of rank %d, int32 of rank 2 expected" % (what, x.dtype, len(n)))
    if n[1] > 1 and s[1] != 1:
        raise ShloError("%s: the last axis is strided" % what)
    return n, s[0]


def rope_noalloc(x, positions, phases, out, *, interleaved=False, inverse=False, factor=1.0, stream=0):
    """x [tokens, heads, dim] turned by positions (int32 [tokens]) into out; phases: rope_phases' on the device."""
    lib = load()
    at = lib.shlo_cuda_device()
    n, xs, dt = _rows(x, "rope: x", at)
    m, ys, dy = _rows(out, "rope: out", at)
    if m != n or dy != dt:
        raise ShloError("rope: out is not x's shape and type")
    t, h, d = n
    if _list(positions, _I32, "rope: positions", at) != t:
        raise ShloError("rope: %d positions for %d tokens" % (positions.shape[0], t))
    check(lib.shlo_rope_noalloc(x.data_ptr(), xs[0], xs[1], positions.data_ptr(), phases.data_ptr(), out.data_ptr(),
                                ys[0], ys[1], t, h, d, 2 * _list(phases, _I64, "rope: phases", at), dt,
                                (1 if interleaved else 0) | (2 if inverse else 0), factor, stream))


class Pool:
    """A paged cache over the caller's tensors: k and v int8 [pages, heads, page_tokens, head_dim] (any strides but
    the last axis's, the same for both), their scales float32 [pages, heads]. Holds on to the tensors."""

    __slots__ = ("c", "keep", "device")

    def __init__(self, k, v, k_scale, v_scale):
        n, m, s, z = k.shape, k_scale.shape, k.stride(), k_scale.stride()
        at = self.device = k.get_device() if hasattr(k, "get_device") else None
        if not k.is_cuda:
            _elsewhere(k, at)
        if _code(k, at) != _I8 or _code(v, at) != _I8 or len(n) != 4:
            raise ShloError("cache: k and v are int8 [pages, heads, page_tokens, head_dim]")
        if v.shape != n or v.stride() != s or s[3] != 1:
            raise ShloError("cache: k and v differ in shape or strides, or their last axis is strided")
        if _code(k_scale, at) != _F32 or _code(v_scale, at) != _F32 or m != n[:2] or v_scale.shape != m or v_scale.stride() != z:
            raise ShloError("cache: the scales are not float32 [pages, heads] with the same strides")
        self.keep = (k, v, k_scale, v_scale)
        self.c = KvPool(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n[0], s[0], s[1], s[2],
                        z[0], z[1], n[1], n[3], n[2])


def _pool(pool, at):
    if pool.device is not None:
        raise ShloError("a cache on device %d, but device %d is the current one" % (pool.device, at))


def _batch(starts, lens, tables, tokens, at):
    (n, w), stride = _tables(tables, "batch: tables", at)
    a, b = _list(starts, _I32, "batch: starts", at), _list(lens, _I32, "batch: lens", at)
    if a != n + 1 or b != n:
        raise ShloError("batch: %d starts and %d lengths for tables of %d sequences" % (a, b, n))
    return KvBatch(starts.data_ptr(), lens.data_ptr(), tables.data_ptr(), stride, n, w, tokens)


def append_noalloc(pool: Pool, k, v, starts, lens, tables, *, stream=0):
    """k and v [tokens, heads, dim] rounded into the pages of their sequences."""
    lib = load()
    at = lib.shlo_cuda_device()
    n, ks, dt = _rows(k, "kv_append: k", at)
    m, vs, dv = _rows(v, "kv_append: v", at)
    c = pool.c
    if pool.device != at:
        _pool(pool, at)
    if m != n or dv != dt or n[1] != c.heads or n[2] != c.head_dim:
        raise ShloError("kv_append: k and v are not [tokens, %d, %d] of one type" % (c.heads, c.head_dim))
    check(lib.shlo_kv_append_noalloc(c, _batch(starts, lens, tables, n[0], at), k.data_ptr(), ks[0], ks[1], v.data_ptr(),
                                     vs[0], vs[1], dt, stream))


def gather_noalloc(pool: Pool, tables, seq, pos, k, v, *, stream=0):
    """The cache's values of tokens (seq[i], pos[i]) into k and v [n, heads, dim]."""
    lib = load()
    at = lib.shlo_cuda_device()
    n, ks, dt = _rows(k, "kv_gather: k", at)
    m, vs, dv = _rows(v, "kv_gather: v", at)
    (seqs, width), stride = _tables(tables, "kv_gather: tables", at)
    c, t = pool.c, _list(seq, _I32, "kv_gather: seq", at)
    if pool.device != at:
        _pool(pool, at)
    if _list(pos, _I32, "kv_gather: pos", at) != t or n != (t, c.heads, c.head_dim) or m != n or dv != dt:
        raise ShloError("kv_gather: pos, k and v are not of %d tokens, %d heads of %d" % (t, c.heads, c.head_dim))
    check(lib.shlo_kv_gather_noalloc(c, tables.data_ptr(), stride, seqs, width, seq.data_ptr(), pos.data_ptr(), t,
                                     k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], dt, stream))


def attend_workspace() -> int:
    """Bytes of the workspace that attend_noalloc needs on the current device; zero it once."""
    n = ctypes.c_size_t()
    check(load().shlo_kv_attend_workspace(ctypes.byref(n)))
    return n.value


def attend_noalloc(pool: Pool, q, starts, lens, tables, out, *, workspace, scale, lse=None, causal=True, window=0,
                   stream=0):
    """q [tokens, query heads, dim] against the cache into out (and lse, float32 [tokens, query heads])."""
    lib = load()
    at = lib.shlo_cuda_device()
    n, qs, dt = _rows(q, "kv_attend: q", at)
    m, os_, do = _rows(out, "kv_attend: out", at)
    t, h, d = n
    c = pool.c
    if pool.device != at:
        _pool(pool, at)
    if d != c.head_dim:
        raise ShloError("kv_attend: queries of width %d, the cache's heads are %d wide" % (d, c.head_dim))
    if m != n or do != dt:
        raise ShloError("kv_attend: out is not q's shape and type")
    lp = None
    try:
        if workspace.get_device() != at:
            _elsewhere(workspace, at)
    except AttributeError:
        _elsewhere(workspace, at)
    if lse is not None:
        if _code(lse, at) != _F32 or lse.shape != (t, h) or (t and h and not lse.is_contiguous()):
            raise ShloError("kv_attend: lse is not a contiguous float32 [%d, %d]" % (t, h))
        lp = lse.data_ptr()
    check(lib.shlo_kv_attend_noalloc(c, _batch(starts, lens, tables, t, at), q.data_ptr(), qs[0], qs[1], h, dt, scale,
                                     1 if causal else 0, window, out.data_ptr(), os_[0], os_[1], lp,
                                     workspace.data_ptr(), workspace.numel() * workspace.element_size(), stream))


# ---- on arrays (mlx.Arr), in the library's own memory ----

def rope(x: M.Arr, positions: M.Arr, phases: M.Arr, *, interleaved=False, inverse=False, factor=1.0) -> M.Arr:
    """x [tokens, heads, dim] turned by positions (int32 [tokens]); phases: rope_phases' as an int64 array. May be
    called inside a compiled function."""
    t, h, d = M.shape(x)
    words = [t, h, d, 2 * M.shape(phases)[0], (1 if interleaved else 0) | (2 if inverse else 0),
             int(np.array([factor], np.float32).view(np.uint32)[0])]
    return M.kernel_apply(Run.kernel("rope"), [x, positions, phases, Run.params(words)], [[t, h, d]],
                          bytes([M.dtype(x)]), [max(t, 1), 1, 1], [64, 1, 1])[0]


class Cache:
    """A paged key/value cache in 8 bits in the library's memory (shlo_kv_new). Which pages a sequence has is the
    caller's to say, in the tables; not for compiled functions."""

    __slots__ = ("h", "heads", "head_dim", "page_tokens", "pages")

    def __init__(self, pages: int, heads: int, head_dim: int, page_tokens: int = 64):
        h = ctypes.c_void_p()
        check(load().shlo_kv_new(pages, heads, head_dim, page_tokens, ctypes.byref(h)))
        self.h = h.value
        self.pages, self.heads, self.head_dim, self.page_tokens = pages, heads, head_dim, page_tokens

    def __del__(self):
        h = getattr(self, "h", None)
        if h:
            try:
                load().shlo_kv_free(h)
            except Exception:
                pass
            self.h = None

    def storage(self) -> KvPool:
        p = KvPool()
        check(load().shlo_kv_storage(self.h, p))
        return p

    def append(self, k: M.Arr, v: M.Arr, starts: M.Arr, lens: M.Arr, tables: M.Arr) -> None:
        check(load().shlo_kv_append(self.h, k.h, v.h, starts.h, lens.h, tables.h))

    def gather(self, tables: M.Arr, seq: M.Arr, pos: M.Arr, dtype: int = M.dtF32):
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        check(load().shlo_kv_gather(self.h, tables.h, seq.h, pos.h, dtype, ctypes.byref(k), ctypes.byref(v)))
        return M.Arr(k.value), M.Arr(v.value)

    def attend(self, q: M.Arr, starts: M.Arr, lens: M.Arr, tables: M.Arr, *, scale: float, causal=True, window=0,
               lse=False):
        """The attention's result, or (result, lse)."""
        o, l = ctypes.c_void_p(), ctypes.c_void_p()
        check(load().shlo_kv_attend(self.h, q.h, starts.h, lens.h, tables.h, scale, 1 if causal else 0, window,
                                    ctypes.byref(o), ctypes.byref(l) if lse else None))
        return (M.Arr(o.value), M.Arr(l.value)) if lse else M.Arr(o.value)
