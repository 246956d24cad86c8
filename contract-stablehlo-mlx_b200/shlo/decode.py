"""The decoder operators: rotary positions (with the norm of queries and keys), the
paged key/value cache in 8 bits and the attention that reads it, products in 8-bit
integers, and beam search, for hosts that generate token by token.

The *_noalloc functions take device tensors of the caller's own -- objects with
data_ptr(), shape, stride(), dtype, is_cuda, numel(), element_size() and is_contiguous(), as
a torch.Tensor has them; nothing here imports torch -- and queue their work on `stream` (a cudaStream_t as
an integer; 0 is the default stream) of the device that is current in CUDA. A tensor of another device is refused,
as far as it says where it lies (get_device()). They allocate nothing. Every one is one call
of include/shlo_cuda.h, whose comments say what it computes; errors raise ShloError.
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np

from . import mlx as M
from . import run as Run
from ._lib import BEAM_ARGS, KV_FORK_ARGS, MUL_MAT8_ARGS, NORM_ROPE_ARGS, KvBatch, KvPool, ShloError, check, load

_UNPACKED = (struct.error, OverflowError)  # a number that a descriptor's field does not hold
_norm_rope, _mul_mat8, _beam, _fork = NORM_ROPE_ARGS.pack, MUL_MAT8_ARGS.pack, BEAM_ARGS.pack, KV_FORK_ARGS.pack


def _words(what, *numbers):
    """Numbers that go as 32-bit arguments, which would be cut to what fits."""
    for v in numbers:
        if not -1 << 31 <= v < 1 << 31:
            raise ShloError("%s: %d is no 32-bit number" % (what, v))


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


def _workspace(x, at):
    """A workspace's pointer and its bytes."""
    if x is None:
        return 0, 0
    try:
        if x.get_device() != at:
            _elsewhere(x, at)
    except AttributeError:
        _elsewhere(x, at)
    if not x.is_contiguous():  # (its values are fewer bytes, or others, than it names)
        raise ShloError("a workspace that is not contiguous")
    return x.data_ptr(), x.numel() * x.element_size()


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
    wp, wn = _workspace(workspace, at)
    if lse is not None:
        if _code(lse, at) != _F32 or lse.shape != (t, h) or (t and h and not lse.is_contiguous()):
            raise ShloError("kv_attend: lse is not a contiguous float32 [%d, %d]" % (t, h))
        lp = lse.data_ptr()
    check(lib.shlo_kv_attend_noalloc(c, _batch(starts, lens, tables, t, at), q.data_ptr(), qs[0], qs[1], h, dt, scale,
                                     1 if causal else 0, window, out.data_ptr(), os_[0], os_[1], lp,
                                     wp, wn, stream))


def _weights(q_weight, k_weight, q_heads, h, d, what, at):
    """The two weights' pointers and their type."""
    if not 0 <= q_heads <= h:
        raise ShloError("%s: %d query heads of %d" % (what, q_heads, h))
    code, q, k = _F32, 0, 0
    if q_weight is not None:
        code, q = _vector(q_weight, d, what + ": q_weight", at)
    if k_weight is not None:
        c, k = _vector(k_weight, d, what + ": k_weight", at)
        if q and c != code:
            raise ShloError("%s: weights of two types" % what)
        code = c
    return q, k, code


def _vector(w, d, what, at):
    c = _code(w, at)
    if c != _F16 and c != _F32 or w.shape != (d,) or (d > 1 and w.stride()[0] != 1):
        raise ShloError("%s is not a contiguous float16 or float32 [%d]" % (what, d))
    return c, w.data_ptr()


def norm_rope_noalloc(x, positions, phases, out, *, q_heads, q_weight, k_weight, eps, interleaved=False, factor=1.0,
                      stream=0):
    """x [tokens, heads, dim], each head normed (by the root of its mean square), weighted -- the first q_heads by
    q_weight, the others by k_weight, [dim], None for ones -- and turned by positions into out."""
    lib = load()
    at = lib.shlo_cuda_device()
    n, xs, dt = _rows(x, "norm_rope: x", at)
    m, ys, dy = _rows(out, "norm_rope: out", at)
    if m != n or dy != dt:
        raise ShloError("norm_rope: out is not x's shape and type")
    t, h, d = n
    if _list(positions, _I32, "norm_rope: positions", at) != t:
        raise ShloError("norm_rope: %d positions for %d tokens" % (positions.shape[0], t))
    wq, wk, dw = _weights(q_weight, k_weight, q_heads, h, d, "norm_rope", at)
    try:
        if lib.shlo_norm_rope_noalloc(
                _norm_rope(x.data_ptr(), xs[0], xs[1], positions.data_ptr(), phases.data_ptr(), wq, wk, out.data_ptr(), ys[0],
                           ys[1], 0, 0, 0, 0, 0, 0, 0, t, h, d, 2 * _list(phases, _I64, "norm_rope: phases", at), q_heads, eps,
                           factor, 1 if interleaved else 0, dt, dw), stream):
            check(1)
    except _UNPACKED as e:
        raise ShloError("norm_rope: %s" % e) from None


def norm_rope_workspace() -> int:
    """Bytes of the workspace that norm_rope_grad_noalloc needs on the current device."""
    n = ctypes.c_size_t()
    check(load().shlo_norm_rope_workspace(ctypes.byref(n)))
    return n.value


def norm_rope_grad_noalloc(x, dy, positions, phases, dx, dq_weight=None, dk_weight=None, *, q_heads, q_weight, k_weight,
                           eps, workspace=None, interleaved=False, factor=1.0, stream=0):
    """The gradient of norm_rope_noalloc: of its output dy, into dx and the weights' (float32 [dim], None where they are
    not asked for)."""
    lib = load()
    at = lib.shlo_cuda_device()
    n, xs, dt = _rows(x, "norm_rope_grad: x", at)
    m, gs, dg = _rows(dy, "norm_rope_grad: dy", at)
    o, ys, do = _rows(dx, "norm_rope_grad: dx", at)
    if m != n or dg != dt or o != n or do != dt:
        raise ShloError("norm_rope_grad: dy or dx is not x's shape and type")
    t, h, d = n
    if _list(positions, _I32, "norm_rope_grad: positions", at) != t:
        raise ShloError("norm_rope_grad: %d positions for %d tokens" % (positions.shape[0], t))
    wq, wk, dw = _weights(q_weight, k_weight, q_heads, h, d, "norm_rope_grad", at)
    sums = [0, 0]
    for i, w in enumerate((dq_weight, dk_weight)):
        if w is not None:
            if _code(w, at) != _F32 or w.shape != (d,) or (d > 1 and w.stride()[0] != 1):
                raise ShloError("norm_rope_grad: a weight's gradient is not a contiguous float32 [%d]" % d)
            sums[i] = w.data_ptr()
    wp, wn = _workspace(workspace, at)
    try:
        if lib.shlo_norm_rope_grad_noalloc(
                _norm_rope(x.data_ptr(), xs[0], xs[1], positions.data_ptr(), phases.data_ptr(), wq, wk, dx.data_ptr(), ys[0],
                           ys[1], dy.data_ptr(), gs[0], gs[1], sums[0], sums[1], wp, wn, t, h, d,
                           2 * _list(phases, _I64, "norm_rope_grad: phases", at), q_heads, eps, factor, 1 if interleaved else 0,
                           dt, dw), stream):
            check(1)
    except _UNPACKED as e:
        raise ShloError("norm_rope_grad: %s" % e) from None


# ---- products in 8-bit integers ----

def _matrix(x, codes, what, at):
    """[rows, n] whose last axis is contiguous, of one of the types: (rows, n, row stride, type code)."""
    c, n, s = _code(x, at), x.shape, x.stride()
    if c not in codes or len(n) != 2:
        raise ShloError("%s: %s of rank %d not carried" % (what, x.dtype, len(n)))
    if n[1] > 1 and s[1] != 1:
        raise ShloError("%s: the last axis is strided" % what)
    return n[0], n[1], s[0], c


def _scales(x, n, what, at):
    if _code(x, at) != _F32 or x.shape != (n,) or (n > 1 and x.stride()[0] != 1):
        raise ShloError("%s is not a contiguous float32 [%d]" % (what, n))
    return x.data_ptr()


def quantise_rows_noalloc(x, q, scale, *, stream=0):
    """x [rows, n] rounded to int8 row by row into q, by scale (float32 [rows]); weights [channels, n] too."""
    lib = load()
    at = lib.shlo_cuda_device()
    r, n, xs, dt = _matrix(x, (_F16, _F32), "quantise_rows: x", at)
    rq, nq, qs, _ = _matrix(q, (_I8,), "quantise_rows: q", at)
    if (rq, nq) != (r, n):
        raise ShloError("quantise_rows: q is not x's shape")
    if r > 1 and qs < n:
        raise ShloError("quantise_rows: rows of q overlap")
    _words("quantise_rows", n)
    check(lib.shlo_quantise_rows_noalloc(x.data_ptr(), xs, r, n, dt, q.data_ptr(), qs, _scales(scale, r, "quantise_rows: scale", at),
                                         stream))


def _product(entry, x, xs, x_scale, r, n, x_dtype, w, w_scale, out, bias, wp, wn, what, at, stream):
    m, nw, ws, _ = _matrix(w, (_I8,), what + ": w", at)
    ro, mo, ys, dt = _matrix(out, (_F16, _F32), what + ": out", at)
    if nw != n or ro != r or mo != m:
        raise ShloError("%s: [%d, %d] by weights [%d, %d] into [%d, %d]" % (what, r, n, m, nw, ro, mo))
    if r > 1 and ys < m:
        raise ShloError("%s: rows of out overlap" % what)
    try:
        if entry(_mul_mat8(x.data_ptr(), xs, x_scale, w.data_ptr(), ws, _scales(w_scale, m, what + ": w_scale", at),
                           0 if bias is None else _scales(bias, m, what + ": bias", at), out.data_ptr(), ys, wp, wn, r, n, m, dt,
                           x_dtype), stream):
            check(1)
    except _UNPACKED as e:
        raise ShloError("%s: %s" % (what, e)) from None


def mul_mat8_noalloc(x, x_scale, w, w_scale, out, *, bias=None, stream=0):
    """x int8 [rows, n] by weights int8 [channels, n], times both scales, + bias (float32 [channels]) into out
    (float16 or float32 [rows, channels]). Rows of x and w begin on multiples of 16 bytes."""
    lib = load()
    at = lib.shlo_cuda_device()
    r, n, xs, _ = _matrix(x, (_I8,), "mul_mat8: x", at)
    _product(lib.shlo_mul_mat8_noalloc, x, xs, _scales(x_scale, r, "mul_mat8: x_scale", at), r, n, _I8, w, w_scale, out, bias, 0,
             0, "mul_mat8", at, stream)


def linear8_workspace(rows: int, n: int) -> int:
    """Bytes of the workspace that linear8_noalloc needs for so many rows of n values."""
    _words("linear8_workspace", n)
    b = ctypes.c_size_t()
    check(load().shlo_linear8_workspace(rows, n, ctypes.byref(b)))
    return b.value


def linear8_noalloc(x, w, w_scale, out, *, workspace, bias=None, stream=0):
    """x [rows, n] (float16 or float32) rounded to 8 bits row by row, by weights int8 [channels, n] as mul_mat8_noalloc."""
    lib = load()
    at = lib.shlo_cuda_device()
    r, n, xs, dt = _matrix(x, (_F16, _F32), "linear8: x", at)
    wp, wn = _workspace(workspace, at)
    _product(lib.shlo_linear8_noalloc, x, xs, 0, r, n, dt, w, w_scale, out, bias, wp, wn, "linear8", at, stream)


# ---- beam search ----

def _grid(x, code, shape, what, at):
    if _code(x, at) != code or x.shape != shape or not x.is_contiguous():
        raise ShloError("%s is not a contiguous %s [%d, %d]" % ((what, "float32" if code == _F32 else "int32") + shape))
    return x.data_ptr()


def beam_workspace(seqs: int, beams: int, keep: int, vocab: int) -> int:
    """Bytes of the workspace that beam_select_noalloc needs."""
    _words("beam_workspace", seqs, beams, keep, vocab)
    n = ctypes.c_size_t()
    check(load().shlo_beam_workspace(seqs, beams, keep, vocab, ctypes.byref(n)))
    return n.value


def beam_select_noalloc(logits, scores, next_scores, parents, tokens, *, workspace, ended=None, end_token=-1, stream=0):
    """The best continuations of every sequence's beams: logits [seqs * beams, vocab], scores float32 [seqs, beams] ->
    next_scores float32, parents (rows of the logits) and tokens int32, each [seqs, keep]. ended int32 [seqs, beams]."""
    lib = load()
    at = lib.shlo_cuda_device()
    rows, vocab, stride, dt = _matrix(logits, (_F16, _F32), "beam_select: logits", at)
    if len(scores.shape) != 2 or len(next_scores.shape) != 2:
        raise ShloError("beam_select: scores and next_scores are of rank 2")
    (seqs, beams), keep = scores.shape, next_scores.shape[1]
    if rows != seqs * beams:
        raise ShloError("beam_select: %d rows of logits for %d sequences of %d beams" % (rows, seqs, beams))
    wp, wn = _workspace(workspace, at)
    try:
        if lib.shlo_beam_select_noalloc(
                _beam(logits.data_ptr(), stride, _grid(scores, _F32, (seqs, beams), "beam_select: scores", at),
                      0 if ended is None else _grid(ended, _I32, (seqs, beams), "beam_select: ended", at),
                      _grid(next_scores, _F32, (seqs, keep), "beam_select: next_scores", at),
                      _grid(parents, _I32, (seqs, keep), "beam_select: parents", at),
                      _grid(tokens, _I32, (seqs, keep), "beam_select: tokens", at), wp, wn, seqs, beams, keep, vocab, end_token, dt),
                stream):
            check(1)
    except _UNPACKED as e:
        raise ShloError("beam_select: %s" % e) from None


def fork_noalloc(pool: Pool, tables, lens, parents, fresh, out_tables, out_lens, *, stream=0):
    """Row r of the new tables and lengths goes on from row parents[r] (-1: none) of the old ones; a last page that is
    not full is copied into page fresh[r] for all but the first row that continues its owner."""
    lib = load()
    at = lib.shlo_cuda_device()
    (rows, width), stride = _tables(tables, "kv_fork: tables", at)
    (news, w), ostride = _tables(out_tables, "kv_fork: out_tables", at)
    if pool.device != at:
        _pool(pool, at)
    # (a selection's parents come as [sequences, beams])
    n = parents.shape
    flat = n[0] if len(n) == 1 else parents.numel() if len(n) and parents.is_contiguous() else -1
    if _code(parents, at) != _I32 or flat != news or (len(n) == 1 and news > 1 and parents.stride()[0] != 1):
        raise ShloError("kv_fork: parents are not int32 of %d rows" % news)
    if w != width or _list(lens, _I32, "kv_fork: lens", at) != rows or _list(fresh, _I32, "kv_fork: fresh", at) != news or \
            _list(out_lens, _I32, "kv_fork: out_lens", at) != news:
        raise ShloError("kv_fork: lens, fresh, out_tables and out_lens are not of %d rows continued by %d, tables of %d pages"
                        % (rows, news, width))
    if news > 1 and ostride < width:
        raise ShloError("kv_fork: rows of out_tables overlap")
    try:
        if lib.shlo_kv_fork_noalloc(
                pool.c, _fork(tables.data_ptr(), lens.data_ptr(), stride, parents.data_ptr(), fresh.data_ptr(), out_tables.data_ptr(),
                              out_lens.data_ptr(), ostride, rows, news, width), stream):
            check(1)
    except _UNPACKED as e:
        raise ShloError("kv_fork: %s" % e) from None


# ---- on arrays (mlx.Arr), in the library's own memory ----

def _bits(x: float) -> int:
    return int(np.array([x], np.float32).view(np.uint32)[0])


def rope(x: M.Arr, positions: M.Arr, phases: M.Arr, *, interleaved=False, inverse=False, factor=1.0) -> M.Arr:
    """x [tokens, heads, dim] turned by positions (int32 [tokens]); phases: rope_phases' as an int64 array. May be
    called inside a compiled function."""
    t, h, d = M.shape(x)
    words = [t, h, d, 2 * M.shape(phases)[0], (1 if interleaved else 0) | (2 if inverse else 0),
             _bits(factor)]
    return M.kernel_apply(Run.kernel("rope"), [x, positions, phases, Run.params(words)], [[t, h, d]],
                          bytes([M.dtype(x)]), [max(t, 1), 1, 1], [64, 1, 1])[0]


def norm_rope(x: M.Arr, positions: M.Arr, phases: M.Arr, q_weight: M.Arr, k_weight: M.Arr, *, q_heads: int, eps: float,
              interleaved=False, factor=1.0) -> M.Arr:
    """x [tokens, heads, dim], each head normed, weighted (the first q_heads by q_weight, the others by k_weight, [dim])
    and turned by positions. May be called inside a compiled function, as may what follows up to Cache."""
    t, h, d = M.shape(x)
    if not 0 <= q_heads <= h:
        raise ShloError("norm_rope: %d query heads of %d" % (q_heads, h))
    words = [t, h, d, 2 * M.shape(phases)[0], 1 if interleaved else 0, _bits(factor), q_heads, _bits(eps)]
    return M.kernel_apply(Run.kernel("norm_rope"), [x, positions, phases, q_weight, k_weight, Run.params(words)], [[t, h, d]],
                          bytes([M.dtype(x)]), [max(t, 1), 1, 1], [64, 1, 1])[0]


def _outs(n):
    return [ctypes.c_void_p() for _ in range(n)]


def norm_rope_grad(x: M.Arr, dy: M.Arr, positions: M.Arr, phases: M.Arr, q_weight: M.Arr, k_weight: M.Arr, *, q_heads: int,
                   eps: float, interleaved=False, factor=1.0):
    """(dx, dq_weight, dk_weight) of norm_rope."""
    _words("norm_rope_grad", q_heads)
    o = _outs(3)
    check(load().shlo_norm_rope_grad(x.h, dy.h, positions.h, phases.h, q_weight.h, k_weight.h, q_heads, eps,
                                     1 if interleaved else 0, factor, *[ctypes.byref(a) for a in o]))
    return tuple(M.Arr(a.value) for a in o)


def quantise_rows(x: M.Arr):
    """(q int8 [rows, n and zeros up to a multiple of 16], scale float32 [rows]) of x [rows, n]."""
    o = _outs(2)
    check(load().shlo_quantise_rows(x.h, *[ctypes.byref(a) for a in o]))
    return tuple(M.Arr(a.value) for a in o)


def linear8(x: M.Arr, w: M.Arr, w_scale: M.Arr, *, x_scale: M.Arr | None = None, bias: M.Arr | None = None,
            dtype: int = M.dtF32) -> M.Arr:
    """x [rows, n] (float, or quantise_rows' with x_scale) by weights (quantise_rows' of [channels, n])."""
    o = ctypes.c_void_p()
    check(load().shlo_linear8(x.h, x_scale.h if x_scale else None, w.h, w_scale.h, bias.h if bias else None, dtype,
                              ctypes.byref(o)))
    return M.Arr(o.value)


def beam_select(logits: M.Arr, scores: M.Arr, keep: int, *, ended: M.Arr | None = None, end_token=-1):
    """(scores, parents, tokens) [sequences, keep] of logits [sequences * beams, vocabulary], scores [sequences, beams]."""
    _words("beam_select", keep, end_token)
    o = _outs(3)
    check(load().shlo_beam_select(logits.h, scores.h, ended.h if ended else None, end_token, keep,
                                  *[ctypes.byref(a) for a in o]))
    return tuple(M.Arr(a.value) for a in o)


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

    def fork(self, tables: M.Arr, lens: M.Arr, parents: M.Arr, fresh: M.Arr):
        """(tables, lens) of the rows that go on from parents; shared last pages are copied into fresh ones."""
        t, l = ctypes.c_void_p(), ctypes.c_void_p()
        check(load().shlo_kv_fork(self.h, tables.h, lens.h, parents.h, fresh.h, ctypes.byref(t), ctypes.byref(l)))
        return M.Arr(t.value), M.Arr(l.value)

    def attend(self, q: M.Arr, starts: M.Arr, lens: M.Arr, tables: M.Arr, *, scale: float, causal=True, window=0,
               lse=False):
        """The attention's result, or (result, lse)."""
        o, l = ctypes.c_void_p(), ctypes.c_void_p()
        check(load().shlo_kv_attend(self.h, q.h, starts.h, lens.h, tables.h, scale, 1 if causal else 0, window,
                                    ctypes.byref(o), ctypes.byref(l) if lse else None))
        return (M.Arr(o.value), M.Arr(l.value)) if lse else M.Arr(o.value)
