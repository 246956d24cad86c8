"""The decoder operators on arrays, and the decoder that runs them together."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import decode_oracle as O  # noqa: E402
from shlo import decode as Dc  # noqa: E402
from shlo import decoder as Dd  # noqa: E402
from shlo import mlx as M  # noqa: E402
from shlo._lib import ShloError  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def device():
    M.set_device(0)


@pytest.mark.parametrize("kind", [np.float16, np.float32])
def test_rope_kernel_on_arrays_and_compiled(kind):
    """The "shlo_rope" kernel on a strided view, called and recorded: the same bits; against the 64-bit form (2^-20
    of the pair's magnitude for the turn, 2^-11 for a float16 result)."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((9, 5, 48)).astype(kind)
    pos = rng.integers(0, 4000, 9).astype(np.int32)
    phases, _ = Dc.rope_phases(32)
    view = M.slice_(M.of_numpy(x), [0, 1, 0], [9, 4, 48], [1, 1, 1])
    args = [view, M.of_numpy(pos), M.of_numpy(phases)]
    got = M.to_numpy(Dc.rope(*args, factor=1.5))
    want = O.rope(x[:, 1:4], pos, 10000.0 ** (-2.0 * np.arange(16) / 32), 1.5)
    tol = 2.0 ** -19 * 1.5 * np.abs(x[:, 1:4].astype(np.float64)).max() + np.abs(want) * (2.0 ** -11 if kind == np.float16 else 0)
    assert np.all(np.abs(got - want) <= tol)
    fn = M.compile_(lambda a: [Dc.rope(*a, factor=1.5)], True)
    for _ in range(2):
        assert M.to_numpy(M.apply(fn, args)[0]).tobytes() == got.tobytes()
    back = M.to_numpy(Dc.rope(Dc.rope(*args), *args[1:], inverse=True))
    assert np.abs(back - x[:, 1:4]).max() < (2e-2 if kind == np.float16 else 1e-5)


def test_rope_kernel_refuses():
    x, pos = M.of_numpy(np.zeros((4, 2, 16), np.float32)), M.of_numpy(np.zeros(4, np.int32))
    phases = M.of_numpy(np.zeros(8, np.int64))
    for args, text in (((x, pos, M.of_numpy(np.zeros(9, np.int64))), "turned"),
                       ((x, M.of_numpy(np.zeros(3, np.int32)), phases), "positions"),
                       ((x, M.of_numpy(np.zeros(4, np.float32)), phases), "int32"),
                       ((x, pos, M.of_numpy(np.zeros(8, np.float32))), "int64"),
                       ((M.of_numpy(np.zeros((4, 2, 16), np.int32)), pos, phases), "not carried")):
        with pytest.raises(ShloError, match=text):
            Dc.rope(*args)


@pytest.mark.parametrize("kind", [np.float16, np.float32])
def test_cache_on_arrays(kind):
    """Append, gather and attend through the handle, on strided views; the cache bit for bit, the attention as the
    pointer form's bound (2^-16 of the largest value, and 2^-10 more for float16 weights and results)."""
    rng = np.random.default_rng(1)
    H, G, D, page, n = 2, 3, 32, 16, 40
    cache = Dc.Cache(8, H, D, page)
    tables = np.array([[3, 1, 5], [7, -1, -1]], np.int32)
    starts, lens = np.array([0, n, n + 5], np.int32), np.array([n, 5], np.int32)
    kv = rng.standard_normal((n + 5, 2 * H + 1, D)).astype(kind)
    q = rng.standard_normal((n + 5, D, H * G)).astype(kind)  # heads innermost: read through a copy
    want = O.Cache(8, H, page, D)
    for a in (want.k, want.v, want.ks, want.vs):
        a[:] = 0
    O.append(want, kv[:, :H], kv[:, H:2 * H], starts, lens, tables)
    arr = M.of_numpy(kv)
    batch = [M.of_numpy(a) for a in (starts, lens, tables)]

    def part(lo, hi):
        return M.slice_(arr, [0, lo, 0], [n + 5, hi, D], [1, 1, 1])
    cache.append(part(0, H), part(H, 2 * H), *batch)
    seq, pos = np.repeat([0, 1], [n, 5]).astype(np.int32), np.concatenate([np.arange(n), np.arange(5)]).astype(np.int32)
    gk, gv = cache.gather(batch[2], M.of_numpy(seq), M.of_numpy(pos), M.dtF32)
    ids = tables[seq, pos // page]
    assert np.array_equal(M.to_numpy(gk), want.k[ids, :, pos % page].astype(np.float32) * want.ks[ids][:, :, None])
    assert np.array_equal(M.to_numpy(gv), want.v[ids, :, pos % page].astype(np.float32) * want.vs[ids][:, :, None])
    out, lse = cache.attend(M.transpose(M.of_numpy(q), [0, 2, 1]), *batch, scale=D ** -0.5, window=20, lse=True)
    wo, wl, mag, vmax = O.attend(want, q.transpose(0, 2, 1), starts, lens, tables, D ** -0.5, True, 20)
    tol = (2.0 ** -16 + (2.0 ** -10 if kind == np.float16 else 0)) * np.maximum(vmax, 1)[..., None]
    assert np.all(np.abs(M.to_numpy(out) - wo) <= tol) and np.abs(M.to_numpy(lse) - wl).max() < 1e-4
    p = cache.storage()
    assert (p.pages, p.heads, p.head_dim, p.page_tokens) == (8, H, D, page) and p.k


def test_cache_refuses():
    for args, text in (((0, 1, 16, 16), "pages"), ((4, 1, 20, 16), "head width"), ((4, 1, 16, 20), "tokens a page"),
                       ((4, 0, 16, 16), "heads")):
        with pytest.raises(ShloError, match=text):
            Dc.Cache(*args)
    cache = Dc.Cache(4, 2, 16, 16)
    z = M.of_numpy(np.zeros((3, 2, 16), np.float32))
    good = [M.of_numpy(a) for a in (np.array([0, 3], np.int32), np.array([3], np.int32), np.zeros((1, 1), np.int32))]
    with pytest.raises(ShloError, match="starts"):
        cache.append(z, z, good[1], good[1], good[2])
    with pytest.raises(ShloError, match="int32"):
        cache.append(z, z, M.of_numpy(np.zeros(2, np.int64)), good[1], good[2])
    with pytest.raises(ShloError, match="not \\[tokens"):
        cache.attend(M.of_numpy(np.zeros((3, 2, 32), np.float32)), *good, scale=1.0)
    with pytest.raises(ShloError, match="multiple"):
        cache.attend(M.of_numpy(np.zeros((3, 3, 16), np.float32)), *good, scale=1.0)
    fn = M.compile_(lambda a: [cache.attend(a[0], *good, scale=1.0)], True)
    with pytest.raises(ShloError, match="compiled function"):
        M.apply(fn, [z])
    cache.append(z, z, *good)  # still usable


def reference(cfg, w, prompts):
    """The decoder in 64 bits, whole sequences at once, keys and values not rounded."""
    from scipy.special import erf
    outs = []
    for x in prompts:
        h = x.astype(np.float64)
        t = len(h)
        freqs = cfg.base ** (-2.0 * np.arange(cfg.dh // 2) / cfg.dh)
        for li in range(cfg.layers):
            p = lambda n: w["l%d_%s" % (li, n)].astype(np.float64)  # noqa: E731

            def norm(a):
                return (a - a.mean(1, keepdims=True)) / np.sqrt(a.var(1, keepdims=True) + 1e-5)
            a = norm(h) * p("g1") + p("b1")
            qkv = (a @ p("wqkv").T + p("cqkv")).reshape(t, -1, cfg.dh)
            q, k, v = np.split(qkv, [cfg.heads, cfg.heads + cfg.kv_heads], 1)
            q, k = O.rope(q, np.arange(t), freqs), O.rope(k, np.arange(t), freqs)
            o = np.zeros_like(q)
            for i in range(cfg.heads):
                g = i // (cfg.heads // cfg.kv_heads)
                s = q[:, i] @ k[:, g].T / math.sqrt(cfg.dh)
                s[np.triu_indices(t, 1)] = -np.inf
                e = np.exp(s - s.max(1, keepdims=True))
                o[:, i] = e / e.sum(1, keepdims=True) @ v[:, g]
            h = h + o.reshape(t, -1) @ p("wo").T + p("co")
            a = norm(h) * p("g2") + p("b2")
            f = a @ p("w1").T + p("c1")
            f = f * 0.5 * (1 + erf(f / math.sqrt(2)))
            h = h + f @ p("w2").T + p("c2")
        outs.append(h)
    return outs


def test_decoder_generates_as_the_whole_sequence():
    """Prompts, then single tokens of several sequences at once, against the 64-bit whole-sequence form. What the
    8-bit cache costs: a value is off by half a step of its page's largest, 1/254 of it, so a head's result by
    about as much of the values' size, and the layer's output adds it through 0.02 weights: 4 % of the outputs'
    spread is allowed for the largest of 50 000 errors, 0.2 % for their mean."""
    cfg = Dd.Config(page_tokens=32)
    w = Dd.init_weights(cfg)
    m = Dd.Decoder(cfg, pages=24, weights=w)
    rng = np.random.default_rng(3)
    xs = [rng.standard_normal((n, cfg.d)).astype(np.float32) for n in (70, 33, 5)]
    want = reference(cfg, w, xs)
    got = [[], [], []]
    a, y = m.start(xs[0][:50])
    got[0].append(y)
    b, y = m.start(xs[1][:10])
    got[1].append(y)
    y = m.step([(a, xs[0][50:60]), (b, xs[1][10:31])])
    got[0].append(y[:10])
    got[1].append(y[10:])
    c, y = m.start(xs[2][:1])
    got[2].append(y)
    for i in range(4):
        news = [(a, xs[0][60 + i:61 + i]), (c, xs[2][1 + i:2 + i])] + ([(b, xs[1][31 + i:32 + i])] if i < 2 else [])
        y = m.step(news)
        got[0].append(y[:1])
        got[2].append(y[1:2])
        if i < 2:
            got[1].append(y[2:])
    got[0].append(m.step([(a, xs[0][64:])]))
    for g, x in zip(got, want):
        g = np.concatenate(g)
        err = np.abs(g - x)
        assert g.shape == x.shape and err.max() < 0.01 * x.std() * 4 and err.mean() < 0.002 * x.std()
    used = 24 - len(m.free)
    m.stop(a)
    assert len(m.free) == 24 - used + 3
    with pytest.raises(ShloError, match="pages"):
        m.start(np.zeros((24 * 32, cfg.d), np.float32))
