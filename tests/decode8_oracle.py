"""Plain 64-bit forms of the norm with rotation, the products in 8 bits, beam search's selection and the cache's
reordering, for their tests: numpy, from the formulas in include/shlo_cuda.h."""
import math

import numpy as np

import decode_oracle as O


def norm_rope(x, positions, freqs, wq, wk, q_heads, eps, factor=1.0, interleaved=False):
    """(y, bound): float64, and of each value the magnitudes that scale its rounding."""
    x = x.astype(np.float64)
    d = x.shape[-1]
    inv = 1.0 / np.sqrt((x * x).sum(-1, keepdims=True) / d + eps)
    w = np.where(np.arange(x.shape[1])[:, None] < q_heads, wq.astype(np.float64), wk.astype(np.float64))
    z = x * inv * w
    return O.rope(z, positions, freqs, factor, interleaved), _pair_sums(np.abs(z), len(freqs), factor, interleaved)


def _pair_sums(m, pairs, factor, interleaved):
    ia = np.arange(0, 2 * pairs, 2) if interleaved else np.arange(pairs)
    ib = ia + 1 if interleaved else ia + pairs
    out = m.copy()
    out[..., ia] = out[..., ib] = factor * (m[..., ia] + m[..., ib])
    return out


def norm_rope_grad(x, dy, positions, freqs, wq, wk, q_heads, eps, factor=1.0, interleaved=False):
    """(dx, its bound, dwq, dwk, their bounds)."""
    x, dy = x.astype(np.float64), dy.astype(np.float64)
    t, h, d = x.shape
    inv = 1.0 / np.sqrt((x * x).sum(-1, keepdims=True) / d + eps)
    w = np.where(np.arange(h)[:, None] < q_heads, wq.astype(np.float64), wk.astype(np.float64))
    n = x * inv
    dz = O.rope(dy, positions, freqs, factor, interleaved, inverse=True)
    mag = _pair_sums(np.abs(dy), len(freqs), factor, interleaved)
    g, gm = dz * w, mag * np.abs(w)
    dx = inv * (g - n * (g * n).mean(-1, keepdims=True))
    bound = inv * (gm + np.abs(n) * (gm * np.abs(n)).mean(-1, keepdims=True))
    s, m = (dz * n).sum(0), (mag * np.abs(n)).sum(0)
    return dx, bound, s[:q_heads].sum(0), s[q_heads:].sum(0), m[:q_heads].sum(0), m[q_heads:].sum(0)


def quantise(x):
    """(q int8, scale float32) of rows: ties by whole-number arithmetic on the values' mantissas."""
    q, scale = np.zeros(x.shape, np.int8), np.zeros(x.shape[0], np.float32)
    for r in range(x.shape[0]):
        v = x[r].astype(np.float64)
        if not np.isfinite(v).all():
            scale[r] = np.nan
            continue
        top = np.abs(v).max()
        scale[r] = np.float32(top) / np.float32(127.0)
        if top == 0:
            continue
        m, e = math.frexp(top)
        b = int(m * 2.0 ** 53)
        for i in np.flatnonzero(v):
            m2, e2 = math.frexp(abs(v[i]))
            # a / top = (int(m2 2^53) / b) 2^(e2 - e)
            num, den = 127 * int(m2 * 2.0 ** 53), b << (e - e2)
            k, rest = divmod(num, den)
            k += 2 * rest > den or (2 * rest == den and k % 2 == 1)
            q[r, i] = k if v[i] > 0 else -k
    return q, scale


def mul_mat8(x, xs, w, ws, bias=None, dtype=np.float32):
    """The stated binary32 operations, in order."""
    acc = x.astype(np.float64) @ w.astype(np.float64).T  # whole numbers below 2^53
    with np.errstate(over="ignore", invalid="ignore"):
        y = acc.astype(np.float32) * xs[:, None] * ws[None, :]
        if bias is not None:
            y = y + bias[None, :]
        return y.astype(dtype)


def beam(z, scores, keep, ended=None, end_token=-1):
    """(scores float64, parents, tokens) [seqs, keep]."""
    seqs, beams = scores.shape
    v = z.shape[1]
    out = np.full((seqs, keep), -np.inf), np.full((seqs, keep), -1, np.int32), np.full((seqs, keep), -1, np.int32)
    for s in range(seqs):
        cand = []
        for b in range(beams):
            row = s * beams + b
            score = float(scores[s, b])
            if ended is not None and ended[s, b]:
                if score > -np.inf:
                    cand.append((-score, b, end_token, row, score))
                continue
            l = z[row].astype(np.float64)
            if np.isnan(l).any() or (l == np.inf).any() or not (l > -np.inf).any() or not score > -np.inf:
                continue
            top = l.max()
            total = score - math.log(math.fsum(np.exp(l - top))) + (l - top)  # (top may be far from 0)
            best = np.lexsort((np.arange(v), -l))[:keep]
            # (a beam's continuations are ordered by their logits)
            cand += [(-total[t], b, int(t), row, total[t]) for t in best if l[t] > -np.inf]
        cand.sort(key=lambda c: c[:3])
        for i, c in enumerate(cand[:keep]):
            out[0][s, i], out[1][s, i], out[2][s, i] = c[4], c[3], c[2]
    return out


def fork(cache, tables, lens, parents, fresh):
    """(tables, lens); the cache's pages are copied in place."""
    page, pages = cache.page, cache.k.shape[0]
    out = np.full((len(parents), tables.shape[1]), -1, np.int32)
    news, seen = np.zeros(len(parents), np.int32), set()
    for r, p in enumerate(parents):
        if not 0 <= p < len(lens):
            continue
        n = news[r] = max(int(lens[p]), 0)
        have = min(-(-n // page), tables.shape[1])
        out[r, :have] = tables[p, :have]
        i, tail = n // page, n % page
        if tail and i < tables.shape[1]:
            old = tables[p, i]
            if p in seen and 0 <= old < pages:
                f = fresh[r]
                out[r, i] = f if 0 <= f < pages else -1
                if 0 <= f < pages:
                    for a in (cache.k, cache.v):
                        a[f, :, :tail] = a[old, :, :tail]
                    for a in (cache.ks, cache.vs):
                        a[f] = a[old]
            seen.add(p)
    return out, news
