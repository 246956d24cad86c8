"""The norm with rotation, the products in 8 bits, beam search and the cache's reordering on arrays, and the decoder that
runs them together."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import decode8_oracle as O8  # noqa: E402
import decode_oracle as O  # noqa: E402
from shlo import decode as Dc  # noqa: E402
from shlo import decoder as Dd  # noqa: E402
from shlo import mlx as M  # noqa: E402
from shlo._lib import ShloError  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def device():
    M.set_device(0)


def arrays(*xs):
    return [M.of_numpy(x) for x in xs]


def rounding(want, kind):
    return np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if kind == np.float16 else 0.0


@pytest.mark.parametrize("kind", [np.float16, np.float32])
def test_norm_rope_on_arrays_and_compiled(kind):
    """On a strided view, called and recorded: the same bits. Tolerances as in tests/test_gpu_decode8.py."""
    rng = np.random.default_rng(0)
    T, H, D, R, HQ = 9, 5, 48, 32, 3
    x, dy = rng.standard_normal((T, H + 1, D)).astype(kind), rng.standard_normal((T, H, D)).astype(kind)
    wq, wk = (1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32)
    pos = rng.integers(0, 4000, T).astype(np.int32)
    freqs = 10000.0 ** (-2.0 * np.arange(R // 2) / R)
    view = M.slice_(M.of_numpy(x), [0, 1, 0], [T, H + 1, D], [1, 1, 1])
    rest = arrays(pos, Dc.rope_phases(R)[0], wq, wk)
    kw = dict(q_heads=HQ, eps=1e-5, factor=1.5)
    got = M.to_numpy(Dc.norm_rope(view, *rest, **kw))
    eps = np.float64(np.float32(1e-5))
    want, mag = O8.norm_rope(x[:, 1:], pos, freqs, wq, wk, HQ, eps, 1.5)
    assert np.all(np.abs(got - want) <= 2.0 ** -19 * mag + rounding(want, kind))
    grads = [M.to_numpy(a) for a in Dc.norm_rope_grad(view, M.of_numpy(dy), *rest, **kw)]
    dx, mag, dq, dk, mq, mk = O8.norm_rope_grad(x[:, 1:], dy, pos, freqs, wq, wk, HQ, eps, 1.5)
    assert np.all(np.abs(grads[0] - dx) <= 2.0 ** -18 * mag + rounding(dx, kind))
    assert np.all(np.abs(grads[1] - dq) <= 2.0 ** -16 * mq) and np.all(np.abs(grads[2] - dk) <= 2.0 ** -16 * mk)
    fn = M.compile_(lambda a: [Dc.norm_rope(a[0], *a[2:], **kw), *Dc.norm_rope_grad(*a, **kw)], True)
    for _ in range(3):
        out = M.apply(fn, [view, M.of_numpy(dy), *rest])
        assert all(M.to_numpy(a).tobytes() == b.tobytes() for a, b in zip(out, [got] + grads))


def test_norm_rope_refuses():
    x, pos, phases, w = arrays(np.zeros((4, 2, 16), np.float32), np.zeros(4, np.int32), np.zeros(8, np.int64), np.ones(16, np.float32))
    for args, kw, text in (((x, pos, M.of_numpy(np.zeros(9, np.int64)), w, w), {}, "turned"),
                           ((x, M.of_numpy(np.zeros(3, np.int32)), phases, w, w), {}, "positions"),
                           ((x, pos, phases, w, M.of_numpy(np.ones(15, np.float32))), {}, "weights"),
                           ((x, pos, phases, w, w), dict(q_heads=3), "query heads"), ((x, pos, phases, w, w), dict(eps=0.0), "eps"),
                           ((M.of_numpy(np.zeros((4, 2, 16), np.int32)), pos, phases, w, w), {}, "not carried")):
        for f in (Dc.norm_rope, lambda a, *b, **k: Dc.norm_rope_grad(a, a, *b, **k)):
            with pytest.raises(ShloError, match=text):
                f(*args, **dict(dict(q_heads=1, eps=1e-6), **kw))


@pytest.mark.parametrize("kind", [np.float16, np.float32])
@pytest.mark.parametrize("r,n,m", [(1, 100, 70), (5, 512, 768), (40, 33, 129)])
def test_linear8_on_arrays_and_compiled(kind, r, n, m):
    rng = np.random.default_rng(n)
    x, w = rng.standard_normal((r, n)).astype(kind), rng.standard_normal((m, n)).astype(np.float32)
    bias = rng.standard_normal(m).astype(np.float32)
    qw, sw = Dc.quantise_rows(M.of_numpy(w))
    q, s = O8.quantise(w)
    pad = np.zeros((m, -(-n // 16) * 16), np.int8)
    pad[:, :n] = q
    assert np.array_equal(M.to_numpy(qw), pad) and M.to_numpy(sw).tobytes() == s.tobytes()
    qx, sx = O8.quantise(x)
    for dt, np_dt in ((M.dtF32, np.float32), (M.dtF16, np.float16)):
        want = O8.mul_mat8(qx, sx, q, s, bias, np_dt).tobytes()
        xa, ba = arrays(x, bias)
        assert M.to_numpy(Dc.linear8(xa, qw, sw, bias=ba, dtype=dt)).tobytes() == want
        a, b = Dc.quantise_rows(xa)
        assert M.to_numpy(Dc.linear8(a, qw, sw, x_scale=b, bias=ba, dtype=dt)).tobytes() == want
        fn = M.compile_(lambda v, dt=dt: [Dc.linear8(v[0], v[1], v[2], bias=v[3], dtype=dt)], True)
        for _ in range(3):
            assert M.to_numpy(M.apply(fn, [xa, qw, sw, ba])[0]).tobytes() == want
    assert M.to_numpy(Dc.linear8(xa, qw, sw)).tobytes() == O8.mul_mat8(qx, sx, q, s).tobytes()


def test_linear8_refuses():
    w, s = Dc.quantise_rows(M.of_numpy(np.ones((6, 20), np.float32)))
    x = M.of_numpy(np.ones((3, 20), np.float32))
    q, t = Dc.quantise_rows(x)
    for f in (lambda: Dc.linear8(M.of_numpy(np.ones((3, 40), np.float32)), w, s), lambda: Dc.linear8(x, w, t), lambda: Dc.linear8(q, w, s),
              lambda: Dc.linear8(x, w, s, x_scale=t), lambda: Dc.linear8(x, w, s, bias=t), lambda: Dc.linear8(x, x, s),
              lambda: Dc.linear8(x, w, s, dtype=M.dtI32), lambda: Dc.quantise_rows(w)):
        with pytest.raises(ShloError):
            f()


@pytest.mark.parametrize("kind", [np.float16, np.float32])
def test_beam_select_on_arrays_and_compiled(kind):
    rng = np.random.default_rng(4)
    z = (rng.standard_normal((6, 3000)) * 2).astype(kind)
    scores, ended = -rng.random((2, 3)).astype(np.float32), np.array([[0, 1, 0], [0, 0, 0]], np.int32)
    want = O8.beam(z, scores, 5, ended, 9)
    fn = M.compile_(lambda v: list(Dc.beam_select(v[0], v[1], 5, ended=v[2], end_token=9)), True)
    for _ in range(2):
        for got in (Dc.beam_select(*arrays(z, scores), 5, ended=M.of_numpy(ended), end_token=9), M.apply(fn, arrays(z, scores, ended))):
            got = [M.to_numpy(a) for a in got]
            assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
            assert np.all(np.abs(got[0] - want[0]) <= 2.0 ** -23 + 2.0 ** -24 * np.abs(want[0]))
    for f in (lambda: Dc.beam_select(*arrays(z, scores.T[:2]), 5), lambda: Dc.beam_select(*arrays(z, scores), 65),
              lambda: Dc.beam_select(*arrays(z, scores), 5, ended=M.of_numpy(scores))):
        with pytest.raises(ShloError):
            f()


def test_fork_on_arrays():
    rng = np.random.default_rng(6)
    H, D, page = 2, 32, 16
    cache, plain = Dc.Cache(12, H, D, page), O.Cache(12, H, page, D)
    for a in (plain.k, plain.v, plain.ks, plain.vs):
        a[:] = 0
    lens, tables = np.array([20, 37], np.int32), np.array([[3, 5, -1], [1, 0, 7]], np.int32)
    starts = np.array([0, 20, 57], np.int32)
    k, v = rng.standard_normal((2, 57, H, D)).astype(np.float32)
    cache.append(*arrays(k, v, starts, lens, tables))
    O.append(plain, k, v, starts, lens, tables)
    parents, fresh = np.array([1, 1, 0, 1, -1], np.int32), np.array([8, 9, 10, 11, -1], np.int32)
    t, n = (M.to_numpy(a) for a in cache.fork(*arrays(tables, lens, parents, fresh)))
    wt, wn = O8.fork(plain, tables, lens, parents, fresh)
    assert np.array_equal(t, wt) and np.array_equal(n, wn)
    seq, pos = np.array([0, 1, 1, 3, 3], np.int32), np.array([36, 33, 5, 36, 20], np.int32)
    got, _ = cache.gather(*arrays(wt, seq, pos))
    want = np.stack([plain.k[wt[s, p // page], :, p % page] * plain.ks[wt[s, p // page]][:, None] for s, p in zip(seq, pos)])
    assert M.to_numpy(got).tobytes() == want.astype(np.float32).tobytes()
    with pytest.raises(ShloError, match="kv_fork"):
        cache.fork(*arrays(tables, lens[:1], parents, fresh))
    with pytest.raises(ShloError, match="compiled"):
        M.apply(M.compile_(lambda a: list(cache.fork(*a)), True), arrays(tables, lens, parents, fresh))


@pytest.mark.parametrize("bits8,norm", [(False, True), (True, False), (True, True)])
def test_decoder_generates_as_the_whole_sequence(bits8, norm):
    """Step by step, several sequences at once, against the whole sequence in one step: both round the same keys and
    values to 8 bits, but a page's scale grows step by step in one and is there at once in the other: a value's second
    rounding is within half a step, 1/254 of its page's largest, and activations' rounding to 8 bits (another half a
    step where a value changes sides) passes such differences on; so a few hundredths of the outputs' size."""
    cfg = Dd.Config(layers=2, d=256, heads=4, kv_heads=2, ffn=512, page_tokens=16, norm_heads=norm, bits8=bits8)
    w = Dd.init_weights(cfg, 5)
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, cfg.d)).astype(np.float32)
    m = Dd.Decoder(cfg, 24, w)
    s, whole = m.start(x)
    a, y = m.start(x[:17])
    b, _ = m.start(x[:3])
    got = [y]
    for i in range(17, 40):
        got.append(m.step([(b, x[i - 14:i - 13]), (a, x[i:i + 1])])[1:])
    assert np.abs(np.concatenate(got) - whole).max() < 0.05 * np.abs(whole).max()


@pytest.mark.parametrize("bits8", [False, True])
def test_search_is_the_one_without_forks(bits8):
    """Against a search whose beams are each begun again from the prompt, one token a step, in caches of their own:
    the same tokens, and scores to 1e-3 (a step's other sequences change how sums are cut, not what is summed)."""
    cfg = Dd.Config(layers=2, d=128, heads=2, kv_heads=1, ffn=256, page_tokens=16, norm_heads=True, bits8=bits8, vocab=301)
    w = Dd.init_weights(cfg, 2)
    m = Dd.Decoder(cfg, 64, w)
    prompt, beams, steps = [5, 17, 200, 3, 9, 120, 44, 7, 1, 250, 12, 13, 14], 3, 8
    got = m.search(prompt, beams, steps)
    assert len(m.free) == 64 and len(got) == beams
    beam = [(0.0, [])]
    for _ in range(steps):
        rows = []
        for _, text in beam:
            s, y = m.start(w["embed"][prompt])
            for t in text:
                y = m.step([(s, w["embed"][[t]])])
            z = m._dense(M.of_numpy(np.ascontiguousarray(y[-1:])), "head", "chead", cfg.vocab, cfg.d, 1)
            rows.append(M.to_numpy(M.reshape(z, [cfg.vocab])).astype(np.float64))
            m.stop(s)
        total = np.concatenate([b[0] + r - r.max() - np.log(np.exp(r - r.max()).sum()) for b, r in zip(beam, rows)])
        best = np.argsort(-total, kind="stable")[:beams]
        beam = [(float(np.float32(total[i])), beam[i // cfg.vocab][1] + [int(i % cfg.vocab)]) for i in best]
    assert [t for _, t in got] == [t for _, t in beam]
    assert np.allclose([a for a, _ in got], [a for a, _ in beam], atol=1e-3)
    ended = m.search(prompt, beams, 30, end=got[0][1][2])  # a token that comes up: beams end at it
    assert len(m.free) == 64 and all(got[0][1][2] not in t[:-1] for _, t in ended)
