"""The decoder operators: rotary positions, the paged key/value cache in 8 bits and
the attention that reads it, for hosts that generate token by token.

The *_noalloc functions take device tensors of the caller's own -- objects with
data_ptr(), shape, stride(), dtype and element_size(), as a torch.Tensor has them;
nothing here imports torch -- and queue their work on `stream` (a cudaStream_t as
an integer; 0 is the default stream). They allocate nothing. Every one is one call
of include/shlo_cuda.h, whose comments say what it computes; errors raise ShloError.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import mlx as M
from ._lib import KvBatch, KvPool, ShloError, check, load

SCALINGS = {"none": 0, "linear": 1, "base": 2, "ramp": 3, "blend": 4}

_FLOATS = {"torch.float16": M.dtF16, "torch.float32": M.dtF32}
_I32, _I64, _I8, _F32 = "torch.int32", "torch.int64", "torch.int8", "torch.float32"


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


def _float(x, what):
    t = _FLOATS.get(str(x.dtype))
    if t is None:
        raise ShloError("%s: %s not carried (float16 or float32)" % (what, x.dtype))
    return t


def _want(x, dtype, ndim, what):
    if str(x.dtype) != dtype or len(x.shape) != ndim:
        raise ShloError("%s: %s of rank %d, %s of rank %d expected" % (what, x.dtype, len(x.shape), dtype, ndim))


def _packed(x, what):
    """The last axis's values are contiguous."""
    if x.shape[-1] > 1 and x.stride()[-1] != 1:
        raise ShloError("%s: the last axis is strided" % what)


def _rows(x, what):
    """[tokens, heads, dim]: its token and head strides."""
    if len(x.shape) != 3:
        raise ShloError("%s: rank %d, [tokens, heads, dim] expected" % (what, len(x.shape)))
    _packed(x, what)
    s = x.stride()
    return s[0], s[1]


def rope_noalloc(x, positions, phases, out, *, interleaved=False, inverse=False, factor=1.0, stream=0):
    """x [tokens, heads, dim] turned by positions (int32 [tokens]) into out; phases: rope_phases' on the device."""
    dt = _float(x, "rope")
    xs, ys = _rows(x, "rope: x"), _rows(out, "rope: out")
    t, h, d = x.shape
    if tuple(out.shape) != (t, h, d) or str(out.dtype) != str(x.dtype):
        raise ShloError("rope: out is not x's shape and type")
    _want(positions, _I32, 1, "rope: positions")
    _want(phases, _I64, 1, "rope: phases")
    _packed(positions, "rope: positions")
    _packed(phases, "rope: phases")
    if positions.shape[0] != t:
        raise ShloError("rope: %d positions for %d tokens" % (positions.shape[0], t))
    check(load().shlo_rope_noalloc(x.data_ptr(), xs[0], xs[1], positions.data_ptr(), phases.data_ptr(), out.data_ptr(),
                                   ys[0], ys[1], t, h, d, 2 * phases.shape[0], dt,
                                   (1 if interleaved else 0) | (2 if inverse else 0), factor, stream))


class Pool:
    """A paged cache over the caller's tensors: k and v int8 [pages, heads, page_tokens, head_dim] (any strides but
    the last axis's, the same for both), their scales float32 [pages, heads]. Holds on to the tensors."""

    __slots__ = ("c", "keep")

    def __init__(self, k, v, k_scale, v_scale):
        for x, what in ((k, "cache: k"), (v, "cache: v")):
            _want(x, _I8, 4, what)
            _packed(x, what)
        for x, what in ((k_scale, "cache: k_scale"), (v_scale, "cache: v_scale")):
            _want(x, _F32, 2, what)
        p, h, t, d = k.shape
        s, z = k.stride(), k_scale.stride()
        if tuple(v.shape) != (p, h, t, d) or tuple(v.stride()) != tuple(s):
            raise ShloError("cache: k and v differ in shape or strides")
        if tuple(k_scale.shape) != (p, h) or tuple(v_scale.shape) != (p, h) or tuple(v_scale.stride()) != tuple(z):
            raise ShloError("cache: the scales are not [pages, heads] with the same strides")
        self.keep = (k, v, k_scale, v_scale)
        self.c = KvPool(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), p, s[0], s[1], s[2], z[0],
                        z[1], h, d, t)


def _batch(starts, lens, tables, tokens):
    _want(starts, _I32, 1, "batch: starts")
    _want(lens, _I32, 1, "batch: lens")
    _want(tables, _I32, 2, "batch: tables")
    _packed(starts, "batch: starts")
    _packed(lens, "batch: lens")
    _packed(tables, "batch: tables")
    n, w = tables.shape
    if starts.shape[0] != n + 1 or lens.shape[0] != n:
        raise ShloError("batch: %d starts and %d lengths for tables of %d sequences" % (starts.shape[0], lens.shape[0], n))
    return KvBatch(starts.data_ptr(), lens.data_ptr(), tables.data_ptr(), tables.stride()[0], n, w, tokens)


def append_noalloc(pool: Pool, k, v, starts, lens, tables, *, stream=0):
    """k and v [tokens, heads, dim] rounded into the pages of their sequences."""
    dt = _float(k, "kv_append")
    ks, vs = _rows(k, "kv_append: k"), _rows(v, "kv_append: v")
    t, h, d = k.shape
    if tuple(v.shape) != (t, h, d) or str(v.dtype) != str(k.dtype) or h != pool.c.heads or d != pool.c.head_dim:
        raise ShloError("kv_append: k and v are not [tokens, %d, %d] of one type" % (pool.c.heads, pool.c.head_dim))
    check(load().shlo_kv_append_noalloc(pool.c, _batch(starts, lens, tables, t), k.data_ptr(), ks[0], ks[1],
                                        v.data_ptr(), vs[0], vs[1], dt, stream))


def gather_noalloc(pool: Pool, tables, seq, pos, k, v, *, stream=0):
    """The cache's values of tokens (seq[i], pos[i]) into k and v [n, heads, dim]."""
    dt = _float(k, "kv_gather")
    ks, vs = _rows(k, "kv_gather: k"), _rows(v, "kv_gather: v")
    _want(tables, _I32, 2, "kv_gather: tables")
    _want(seq, _I32, 1, "kv_gather: seq")
    _want(pos, _I32, 1, "kv_gather: pos")
    for x, what in ((tables, "tables"), (seq, "seq"), (pos, "pos")):
        _packed(x, "kv_gather: " + what)
    n = seq.shape[0]
    shape = (n, pool.c.heads, pool.c.head_dim)
    if pos.shape[0] != n or tuple(k.shape) != shape or tuple(v.shape) != shape or str(v.dtype) != str(k.dtype):
        raise ShloError("kv_gather: pos, k and v are not of %d tokens, %d heads of %d" % shape)
    check(load().shlo_kv_gather_noalloc(pool.c, tables.data_ptr(), tables.stride()[0], tables.shape[0],
                                        tables.shape[1], seq.data_ptr(), pos.data_ptr(), n, k.data_ptr(), ks[0], ks[1],
                                        v.data_ptr(), vs[0], vs[1], dt, stream))


def attend_workspace() -> int:
    """Bytes of the workspace that attend_noalloc needs on the current device; zero it once."""
    n = ctypes.c_size_t()
    check(load().shlo_kv_attend_workspace(ctypes.byref(n)))
    return n.value


def attend_noalloc(pool: Pool, q, starts, lens, tables, out, *, workspace, scale, lse=None, causal=True, window=0,
                   stream=0):
    """q [tokens, query heads, dim] against the cache into out (and lse, float32 [tokens, query heads])."""
    dt = _float(q, "kv_attend")
    qs, os_ = _rows(q, "kv_attend: q"), _rows(out, "kv_attend: out")
    t, h, d = q.shape
    if d != pool.c.head_dim:
        raise ShloError("kv_attend: queries of width %d, the cache's heads are %d wide" % (d, pool.c.head_dim))
    if tuple(out.shape) != (t, h, d) or str(out.dtype) != str(q.dtype):
        raise ShloError("kv_attend: out is not q's shape and type")
    lp = 0
    if lse is not None:
        _want(lse, _F32, 2, "kv_attend: lse")
        if tuple(lse.shape) != (t, h) or (t and h and tuple(lse.stride()) != (h, 1)):
            raise ShloError("kv_attend: lse is not a contiguous [%d, %d]" % (t, h))
        lp = lse.data_ptr()
    check(load().shlo_kv_attend_noalloc(pool.c, _batch(starts, lens, tables, t), q.data_ptr(), qs[0], qs[1], h, dt,
                                        scale, 1 if causal else 0, window, out.data_ptr(), os_[0], os_[1], lp,
                                        workspace.data_ptr(), workspace.numel() * workspace.element_size(), stream))
