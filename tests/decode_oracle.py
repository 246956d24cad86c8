"""Plain 64-bit forms of the decoder operators, for their tests: numpy, one sequence
and one head at a time, from the formulas in include/shlo_cuda.h."""
import math

import numpy as np


def rope(x, positions, freqs, factor=1.0, interleaved=False, inverse=False):
    """x [T, H, D] (any float type) -> float64; freqs in radians a position."""
    x = x.astype(np.float64)
    r = 2 * len(freqs)
    ang = positions.astype(np.float64)[:, None] * np.asarray(freqs, np.float64)[None, :]
    c, s = factor * np.cos(ang)[:, None, :], factor * np.sin(ang)[:, None, :]
    if inverse:
        s = -s
    y = x.copy()
    ia = np.arange(0, r, 2) if interleaved else np.arange(r // 2)
    ib = ia + 1 if interleaved else ia + r // 2
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


class Cache:
    """int8 values [P, H, T, D] and float32 scales [P, H], keys and values alike."""

    def __init__(self, pages, heads, page, dim, seed=0):
        rng = np.random.default_rng(seed)
        shape = (pages, heads, page, dim)
        self.k = np.clip(np.rint(rng.standard_normal(shape) * 36), -127, 127).astype(np.int8)
        self.v = np.clip(np.rint(rng.standard_normal(shape) * 36), -127, 127).astype(np.int8)
        self.ks = (rng.random((pages, heads)) * 0.03 + 0.01).astype(np.float32)
        self.vs = (rng.random((pages, heads)) * 0.03 + 0.01).astype(np.float32)
        self.page = page

    def rows(self, q, s, ids, head):
        """float64 [keys, D] of the pages `ids` (a page outside the cache: zeros)."""
        parts = []
        for i in ids:
            if 0 <= i < q.shape[0]:
                parts.append(q[i, head].astype(np.float64) * np.float64(s[i, head]))
            else:
                parts.append(np.zeros(q.shape[2:], np.float64))
        return np.concatenate(parts) if parts else np.zeros((0, q.shape[3]))


def attend(cache, q, starts, lens, tables, scale, causal=True, window=0):
    """(out, lse, bound): float64, and for each row the sum over its products that
    scales a score's rounding, max |q| . |k| * scale."""
    T, H, D = q.shape
    hk = cache.k.shape[1]
    g = H // hk
    out, lse, mag = np.zeros((T, H, D)), np.full((T, H), -np.inf), np.zeros((T, H))
    vmax = np.zeros((T, H))
    for b in range(len(lens)):
        n = starts[b + 1] - starts[b]
        keys = min(lens[b], tables.shape[1] * cache.page)
        ids = tables[b, :-(-keys // cache.page)]
        at = np.arange(keys)
        there = np.repeat([0 <= i < cache.k.shape[0] for i in ids], cache.page)[:keys].astype(bool) if keys else np.zeros(0, bool)
        for h in range(hk):
            k, v = cache.rows(cache.k, cache.ks, ids, h)[:keys], cache.rows(cache.v, cache.vs, ids, h)[:keys]
            for j in range(n):
                pos = lens[b] - n + j
                seen = there.copy()
                if causal:
                    seen &= at <= pos
                if window:
                    seen &= at > pos - window
                if not seen.any():
                    continue
                for i in range(h * g, (h + 1) * g):
                    qq = q[starts[b] + j, i].astype(np.float64)
                    z = k[seen] @ qq * scale
                    m = z.max()
                    p = np.exp(z - m)
                    out[starts[b] + j, i] = p @ v[seen] / p.sum()
                    lse[starts[b] + j, i] = m + math.log(p.sum()) if np.isfinite(m) else m
                    mag[starts[b] + j, i] = (np.abs(k[seen]) @ np.abs(qq)).max() * abs(scale)
                    vmax[starts[b] + j, i] = np.abs(v[seen]).max()
    return out, lse, mag, vmax


def append(cache, k, v, starts, lens, tables):
    """In place, in the stated binary32 operations."""
    f32 = np.float32
    for x, q, s in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
        x = x.astype(np.float32)
        for b in range(len(lens)):
            n = starts[b + 1] - starts[b]
            first = lens[b] - n
            at = max(first, 0)
            while at < lens[b]:
                i = at // cache.page
                end = min((i + 1) * cache.page, lens[b])
                if i >= tables.shape[1]:
                    break
                p = tables[b, i]
                if 0 <= p < q.shape[0]:
                    old = at - i * cache.page
                    new = x[starts[b] + at - first:starts[b] + end - first]  # [t, H, D]
                    for h in range(q.shape[1]):
                        w = new[:, h]
                        top = f32(np.abs(w).max())
                        sc = top * f32(1.0 / 127.0)
                        if old and (s[p, h] > sc or np.isnan(s[p, h])):
                            sc = s[p, h]
                        if not np.isfinite(w).all():
                            sc = f32(np.nan)
                        if old and sc != s[p, h] and not np.isnan(sc):
                            ratio = s[p, h] / sc if sc > 0 else f32(0)
                            q[p, h, :old] = np.rint(q[p, h, :old].astype(np.float32) * ratio).astype(np.int8)
                        if sc > 0:
                            vals = np.clip(np.rint(w / sc), -127, 127)
                        else:
                            vals = np.zeros_like(w)
                        q[p, h, old:old + end - at] = vals.astype(np.int8)
                        s[p, h] = sc
                at = end
