"""The norm with rotation, the products in 8 bits, beam search's selection and the cache's reordering on the GPU against
plain 64-bit forms (tests/decode8_oracle.py).

Tolerances, from the arithmetic and before any run:
 - norm_rope: a head's mean square is a sum of up to 16 + 5 roundings, 2^-24 each, so its root is within 2^-20; with the
   turn's 2^-20 (|a| + |b|): 2^-19 of those magnitudes; a float16 result adds 2^-11 |y| (2^-25 below its normal range).
 - its gradient: dx is a difference of two such terms, with the sum over a head once more: 2^-18 of the magnitudes; a
   weight's gradient adds the sums over tokens, 256 terms a lane at most here and 100 on the way to the result: 2^-16.
 - quantise_rows, mul_mat8, linear8: bit for bit (the sums are whole numbers, each later step one binary32 operation).
 - beam_select: parents and tokens equal; a score is off by 2^-23 (the terms of the logarithm, each within 2^-24) and its
   own rounding, 2^-24 of it.
 - fork: equal.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import decode8_oracle as O8  # noqa: E402
import decode_oracle as O  # noqa: E402
from shlo import decode as Dc  # noqa: E402
from shlo import mlx as M  # noqa: E402
from shlo._lib import ShloError  # noqa: E402

NP = {"f16": np.float16, "f32": np.float32}
TT = {"f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.set_device(0)
    M.set_device(0)
    yield
    torch.cuda.empty_cache()


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream


def work(n):
    return torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")


# -------------------------------------------------------------- norm_rope ----

def plan(R):
    if not R:
        return np.zeros(0, np.int64), np.zeros(0)
    return Dc.rope_phases(R, 10000.0)[0], 10000.0 ** (-2.0 * np.arange(R // 2) / R)


def rounding(want, kind):
    return np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if kind == "f16" else 0.0


SHAPES = [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 3, 0, 80, 32), (33, 0, 5, 72, 18), (5, 2, 1, 64, 64), (1000, 5, 2, 96, 48),
          (3, 1, 1, 512, 512), (2, 2, 2, 511, 2), (4, 3, 1, 66, 0), (2500, 3, 1, 24, 24), (9, 2, 1, 1, 0), (6, 40, 40, 40, 20)]


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,HQ,HK,D,R", SHAPES)
def test_norm_rope_and_its_gradient(kind, inter, T, HQ, HK, D, R):
    rng = np.random.default_rng(T * 7 + D)
    H = HQ + HK
    x = (rng.standard_normal((T, H, D)) * rng.uniform(0.01, 4, (T, 1, 1))).astype(NP[kind])
    x[0, 0] = 0
    dy = rng.standard_normal((T, H, D)).astype(NP[kind])
    wt = "f32" if T % 2 else kind
    wq, wk = (1 + 0.3 * rng.standard_normal((2, D))).astype(NP[wt])
    pos = rng.integers(-5, 100000, T).astype(np.int32)
    phases, freqs = plan(R)
    args = dict(q_heads=HQ, q_weight=cuda(wq), k_weight=cuda(wk), eps=1e-5, interleaved=inter, factor=1.25, stream=stream())
    out = torch.full((T, H, D), 7.0, dtype=TT[kind], device="cuda")
    Dc.norm_rope_noalloc(cuda(x), cuda(pos), cuda(phases), out, **args)
    eps = np.float64(np.float32(1e-5))
    want, mag = O8.norm_rope(x, pos, freqs, wq, wk, HQ, eps, 1.25, inter)
    assert np.all(np.abs(out.cpu().numpy().astype(np.float64) - want) <= 2.0 ** -19 * mag + rounding(want, kind))

    dw = torch.full((2, D), np.nan, device="cuda")
    w = work(Dc.norm_rope_workspace()).fill_(255)
    Dc.norm_rope_grad_noalloc(cuda(x), cuda(dy), cuda(pos), cuda(phases), out, dw[0], dw[1], workspace=w, **args)
    dx, mag, dq, dk, mq, mk = O8.norm_rope_grad(x, dy, pos, freqs, wq, wk, HQ, eps, 1.25, inter)
    assert np.all(np.abs(out.cpu().numpy().astype(np.float64) - dx) <= 2.0 ** -18 * mag + rounding(dx, kind))
    got = dw.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got[0] - dq) <= 2.0 ** -16 * mq) and np.all(np.abs(got[1] - dk) <= 2.0 ** -16 * mk)
    again, dw2 = torch.empty_like(out), torch.empty_like(dw)
    Dc.norm_rope_grad_noalloc(cuda(x), cuda(dy), cuda(pos), cuda(phases), again, dw2[0], dw2[1], workspace=w, **args)
    assert torch.equal(again, out) and torch.equal(dw, dw2)  # the same call, the same bits
    Dc.norm_rope_grad_noalloc(cuda(x), cuda(dy), cuda(pos), cuda(phases), again.fill_(3.0), **args)  # frozen weights
    assert torch.equal(again, out)


# Heads of nine or ten units (ten lanes), five and six, in float32 or float16, with heads enough for a block's groups; a
# turned part that ends inside a vector.
UNEVEN = [(2500, 3, 2, 80, 32), (9, 20, 4, 72, 24), (9, 30, 10, 40, 40), (7, 30, 6, 48, 48), (9, 8, 40, 80, 80), (700, 30, 7, 96, 96),
          (5, 23, 1, 160, 160), (9, 1, 39, 20, 0), (4000, 0, 3, 72, 72), (2500, 3, 2, 72, 18), (3000, 2, 0, 20, 6), (1300, 5, 1, 66, 34)]


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,HQ,HK,D,R", UNEVEN)
def test_norm_rope_of_heads_that_leave_lanes(kind, inter, T, HQ, HK, D, R):
    test_norm_rope_and_its_gradient(kind, inter, T, HQ, HK, D, R)


def test_norm_rope_of_heads_that_leave_lanes_far_values():
    """float32 heads whose squares leave binary32's range, beside ones whose do not, ten lanes each."""
    rng = np.random.default_rng(8)
    T, H, D, R = 5, 24, 72, 24
    x, dy = rng.standard_normal((2, T, H, D))
    x = (x * np.where(rng.random((T, H, 1)) < 0.3, 1e25, 1.0)).astype(np.float32)
    dy = dy.astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    pos = rng.integers(0, 5000, T).astype(np.int32)
    phases, freqs = plan(R)
    args = dict(q_heads=H, q_weight=cuda(w), k_weight=None, eps=1e-5, stream=stream())
    out = torch.empty(T, H, D, device="cuda")
    Dc.norm_rope_noalloc(cuda(x), cuda(pos), cuda(phases), out, **args)
    eps = np.float64(np.float32(1e-5))
    want, mag = O8.norm_rope(x, pos, freqs, w, w, H, eps)
    assert np.all(np.abs(out.cpu().numpy() - want) <= 2.0 ** -19 * mag)
    Dc.norm_rope_grad_noalloc(cuda(x), cuda(dy), cuda(pos), cuda(phases), out, **args)
    dx, mag = O8.norm_rope_grad(x, dy, pos, freqs, w, w, H, eps)[:2]
    assert np.all(np.abs(out.cpu().numpy() - dx) <= 2.0 ** -18 * mag)


def test_norm_rope_gradient_is_the_differences():
    """<dy, y(x, w)> by central differences of the 64-bit form: a step of 1e-4 leaves 1e-8 of the third derivative
    and 1e-12 of rounding, against 32-bit gradients to 2^-16."""
    rng = np.random.default_rng(5)
    T, H, D, R = 3, 3, 12, 8
    x, dy = rng.standard_normal((T, H, D)).astype(np.float32), rng.standard_normal((T, H, D)).astype(np.float32)
    wq, wk = (1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32)
    pos = rng.integers(0, 500, T).astype(np.int32)
    phases, freqs = plan(R)
    dx, dw = torch.empty(T, H, D, device="cuda"), torch.empty(2, D, device="cuda")
    Dc.norm_rope_grad_noalloc(cuda(x), cuda(dy), cuda(pos), cuda(phases), dx, dw[0], dw[1], q_heads=2, q_weight=cuda(wq),
                              k_weight=cuda(wk), eps=0.1, workspace=work(Dc.norm_rope_workspace()), stream=stream())

    def loss(x, wq, wk):
        return (O8.norm_rope(x, pos, freqs, wq, wk, 2, np.float64(np.float32(0.1)))[0] * dy).sum()
    h = 1e-4
    for got, which in ((dx.cpu().numpy(), 0), (dw[0].cpu().numpy(), 1), (dw[1].cpu().numpy(), 2)):
        for i in np.ndindex(got.shape):
            ops = [a.astype(np.float64) for a in (x, wq, wk)]
            ops[which][i] += h
            up = loss(*ops)
            ops[which][i] -= 2 * h
            assert abs((up - loss(*ops)) / (2 * h) - got[i]) < 1e-5 * max(1.0, np.abs(got).max()) + 1e-6


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_norm_rope_strides_and_in_place(kind):
    """A slice of wider rows at offsets that allow wide loads or none, y in x's place, dx in dy's and in x's."""
    rng = np.random.default_rng(3)
    T, H, D, R = 19, 4, 64, 32
    phases, freqs = plan(R)
    pos = np.arange(T, dtype=np.int32) * 3
    wq, wk = (1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32)
    args = dict(q_heads=3, q_weight=cuda(wq), k_weight=cuda(wk), eps=1e-6, stream=stream())
    for off in (0, 1, 2, 4, 8):
        wide = cuda(rng.standard_normal((T, H + 2, D + 8)).astype(NP[kind]))
        wide_g = cuda(rng.standard_normal((T, H + 1, D + 8)).astype(NP[kind]))
        x, g = wide[:, 1:1 + H, off:off + D], wide_g[:, :H, off:off + D]
        out, dx = torch.empty(T, H, D, dtype=x.dtype, device="cuda"), torch.empty(T, H, D, dtype=x.dtype, device="cuda")
        Dc.norm_rope_noalloc(x, cuda(pos), cuda(phases), out, **args)
        want, mag = O8.norm_rope(x.cpu().numpy(), pos, freqs, wq, wk, 3, np.float64(np.float32(1e-6)))
        assert np.all(np.abs(out.cpu().numpy().astype(np.float64) - want) <= 2.0 ** -19 * mag + rounding(want, kind))
        Dc.norm_rope_grad_noalloc(x, g, cuda(pos), cuda(phases), dx, **args)
        dxw, dmag = O8.norm_rope_grad(x.cpu().numpy(), g.cpu().numpy(), pos, freqs, wq, wk, 3, np.float64(np.float32(1e-6)))[:2]
        assert np.all(np.abs(dx.cpu().numpy().astype(np.float64) - dxw) <= 2.0 ** -18 * dmag + rounding(dxw, kind))
        for place in ("dy", "x"):
            w2, g2 = wide.clone(), wide_g.clone()
            x2, gg = w2[:, 1:1 + H, off:off + D], g2[:, :H, off:off + D]
            to, src, whole = (gg, wide_g, g2) if place == "dy" else (x2, wide, w2)
            Dc.norm_rope_grad_noalloc(x2, gg, cuda(pos), cuda(phases), to, **args)
            assert torch.equal(to, dx)
            to.copy_(g if place == "dy" else x)
            assert torch.equal(whole, src)  # nothing around it was written
        before = wide.clone()
        Dc.norm_rope_noalloc(x, cuda(pos), cuda(phases), x, **args)
        assert torch.equal(x, out)
        x.copy_(before[:, 1:1 + H, off:off + D])
        assert torch.equal(wide, before)


def test_norm_rope_far_values_and_absent_weights():
    """Squares that leave 32 bits' range; NaN and infinity stay in their heads; weights of None are ones."""
    rng = np.random.default_rng(8)
    T, H, D, R = 6, 3, 32, 16
    phases, freqs = plan(R)
    pos = np.arange(T, dtype=np.int32)
    one = np.ones(D, np.float32)
    x = rng.standard_normal((T, H, D)).astype(np.float32)
    x[0] *= 1e30
    x[1] *= 1e-25
    x[2, 0] = 3e38
    x[3, 1] *= 1e19
    dy = rng.standard_normal((T, H, D)).astype(np.float32)
    for eps in (1e-6, 1e-44):
        e = np.float64(np.float32(eps))
        args = dict(q_heads=1, q_weight=None, k_weight=None, eps=eps, stream=stream())
        out, dx = torch.empty(T, H, D, device="cuda"), torch.empty(T, H, D, device="cuda")
        Dc.norm_rope_noalloc(cuda(x), cuda(pos), cuda(phases), out, **args)
        want, mag = O8.norm_rope(x, pos, freqs, one, one, 1, e)
        assert np.all(np.abs(out.cpu().numpy() - want) <= 2.0 ** -19 * mag + 2.0 ** -149)
        Dc.norm_rope_grad_noalloc(cuda(x), cuda(dy), cuda(pos), cuda(phases), dx, **args)
        want, mag = O8.norm_rope_grad(x, dy, pos, freqs, one, one, 1, e)[:2]
        assert np.all(np.abs(dx.cpu().numpy() - want) <= 2.0 ** -18 * mag + 2.0 ** -149)
    y = x.copy()
    y[4, 1, 3] = np.nan
    y[5, 2, 30] = np.inf
    bad = torch.empty(T, H, D, device="cuda")
    Dc.norm_rope_noalloc(cuda(y), cuda(pos), cuda(phases), bad, **args)
    bad, out = bad.cpu().numpy(), out.cpu().numpy()
    assert np.isnan(bad[4, 1]).all() and np.isnan(bad[5, 2, 30])
    bad[4, 1], bad[5, 2] = out[4, 1], out[5, 2]
    assert bad.tobytes() == out.tobytes()


def test_norm_rope_refusals():
    x, pos = torch.zeros(3, 4, 16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    phases, w = torch.zeros(8, dtype=torch.int64, device="cuda"), torch.ones(16, device="cuda")
    kw = dict(q_heads=2, q_weight=w, k_weight=w, eps=1e-6)
    wide = torch.zeros(3, 4, 600, device="cuda")
    for args, change, text in (((x, pos, phases, x[:, :1].expand(3, 4, 16)), {}, "overlap"), ((x, pos, phases, torch.empty_like(x)[:1].expand(3, 4, 16)), {}, "overlap"),
                               ((x, pos, phases, torch.empty_like(x)), dict(eps=0.0), "eps"), ((x, pos, phases, torch.empty_like(x)), dict(eps=float("nan")), "eps"),
                               ((wide, pos, phases, torch.empty_like(wide)), dict(q_weight=None, k_weight=None), "600"),
                               ((x[..., :8], pos, phases, torch.empty_like(x[..., :8])), dict(q_weight=w[:8], k_weight=w[:8]), "turned"),
                               ((x[:2], pos[:2], phases, x[1:]), {}, "overlap")):
        with pytest.raises(ShloError, match=text):
            Dc.norm_rope_noalloc(*args, **dict(kw, **change))
    dx, dw = torch.empty_like(x), torch.empty(2, 16, device="cuda")
    for bad in (None, work(8), work(Dc.norm_rope_workspace() + 8)[4:]):
        with pytest.raises(ShloError, match="workspace"):
            Dc.norm_rope_grad_noalloc(x, x, pos, phases, dx, dw[0], dw[1], workspace=bad, **kw)
    for dq, dk in ((dw[0], dw[0]), (dw.view(-1)[:16], dw.view(-1)[15:31])):
        with pytest.raises(ShloError, match="share memory"):
            Dc.norm_rope_grad_noalloc(x, x, pos, phases, dx, dq, dk, workspace=work(Dc.norm_rope_workspace()), **kw)


def test_norm_rope_broadcast_operands():
    """One head's values for all of them, one token's gradient for all: strides of 0 are read as they are."""
    rng = np.random.default_rng(2)
    T, H, D, R = 6, 4, 32, 32
    phases, freqs = plan(R)
    x, dy = cuda(rng.standard_normal((T, 1, D)).astype(np.float32)).expand(T, H, D), cuda(rng.standard_normal((1, H, D)).astype(np.float32)).expand(T, H, D)
    pos = np.arange(T, dtype=np.int32)
    wq, wk = (1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32)
    kw = dict(q_heads=3, q_weight=cuda(wq), k_weight=cuda(wk), eps=1e-6, stream=stream())
    y, dx, dw = torch.empty(T, H, D, device="cuda"), torch.empty(T, H, D, device="cuda"), torch.empty(2, D, device="cuda")
    Dc.norm_rope_noalloc(x, cuda(pos), cuda(phases), y, **kw)
    Dc.norm_rope_grad_noalloc(x, dy, cuda(pos), cuda(phases), dx, dw[0], dw[1], workspace=work(Dc.norm_rope_workspace()), **kw)
    xn, gn, eps = x.cpu().numpy(), dy.cpu().numpy(), np.float64(np.float32(1e-6))
    want, mag = O8.norm_rope(xn, pos, freqs, wq, wk, 3, eps)
    assert np.all(np.abs(y.cpu().numpy() - want) <= 2.0 ** -19 * mag)
    want, mag, dq, dk, mq, mk = O8.norm_rope_grad(xn, gn, pos, freqs, wq, wk, 3, eps)
    assert np.all(np.abs(dx.cpu().numpy() - want) <= 2.0 ** -18 * mag)
    got = dw.cpu().numpy()
    assert np.all(np.abs(got[0] - dq) <= 2.0 ** -16 * mq) and np.all(np.abs(got[1] - dk) <= 2.0 ** -16 * mk)


def test_norm_rope_no_tokens():
    dw = torch.full((2, 8), 3.0, device="cuda")
    e = torch.empty(0, 2, 8, device="cuda")
    pos, phases = torch.empty(0, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    one = torch.ones(8, device="cuda")
    Dc.norm_rope_noalloc(e, pos, phases, e, q_heads=1, q_weight=one, k_weight=one, eps=1e-6, stream=stream())
    Dc.norm_rope_grad_noalloc(e, e, pos, phases, e, dw[0], dw[1], q_heads=1, q_weight=one, k_weight=one, eps=1e-6,
                              workspace=work(Dc.norm_rope_workspace()), stream=stream())
    assert not dw.any()


# ---------------------------------------------------------------- linear8 ----

def activations(rng, r, n, kind):
    x = (rng.standard_normal((r, n)) * rng.uniform(0.1, 3, (r, 1))).astype(NP[kind])
    if r > 2:
        x[1] = 0
        x[2] = NP[kind](0.75) * rng.integers(-254, 255, n) / 127  # many exact halves of a step
        x[2, 0] = 1.5
    return x


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("r,n", [(1, 1), (3, 7), (5, 64), (4, 1000), (3, 4099), (2, 20000), (300, 33)])
def test_quantise_rows(kind, r, n):
    rng = np.random.default_rng(n)
    x = activations(rng, r, n, kind)
    q, scale = O8.quantise(x)
    for off, pad in ((0, 0), (0, 16), (1, 5)):
        wide = np.full((r, n + pad), 9, x.dtype)
        wide[:, off:off + n] = x
        to = torch.full((r, n + 3), 77, dtype=torch.int8, device="cuda")
        s = torch.empty(r, device="cuda")
        Dc.quantise_rows_noalloc(cuda(wide)[:, off:off + n], to[:, :n], s, stream=stream())
        assert np.array_equal(to[:, :n].cpu().numpy(), q) and s.cpu().numpy().tobytes() == scale.tobytes()
        assert bool((to[:, n:] == 77).all())


def test_quantise_rows_far_values():
    x = np.zeros((9, 40), np.float32)
    rng = np.random.default_rng(1)
    for i, m in enumerate((1e-45, 1e-40, 1e-36, 3e38, 1e30)):
        x[i] = (rng.standard_normal(40) * m * 0.2).astype(np.float32)
        x[i, 3] = m
    x[5, 7], x[6, 8], x[7, 9] = np.nan, np.inf, -np.inf
    x[5:8, 1] = 1.0
    q, scale = O8.quantise(x)
    to, s = torch.empty(9, 40, dtype=torch.int8, device="cuda"), torch.empty(9, device="cuda")
    Dc.quantise_rows_noalloc(cuda(x), to, s, stream=stream())
    assert np.array_equal(to.cpu().numpy(), q)
    assert np.array_equal(s.cpu().numpy(), scale, equal_nan=True)


def weights(rng, m, n):
    pad = -(-n // 16) * 16
    w = rng.integers(-128, 128, (m, pad)).astype(np.int8)  # (what lies behind a row's end is not read as part of it)
    return w, (rng.random(m) * 0.01 + 0.001).astype(np.float32)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("r,n,m", [(1, 1, 1), (1, 512, 768), (1, 4097, 130), (2, 16, 64), (3, 100, 1000), (5, 2000, 129), (8, 640, 257),
                                   (16, 1024, 4096), (17, 515, 300), (24, 4096, 515), (33, 31, 33), (64, 8192, 384), (65, 777, 1001),
                                   (130, 1300, 200), (257, 129, 640), (300, 512, 2050), (1000, 260, 1111), (2, 131071, 3),
                                   (700, 1999, 2049), (2300, 1000, 2700), (100, 200, 40000), (1, 16385, 40),
                                   (1, 70001, 24), (2, 1500, 300), (4, 509, 1300), (4, 6145, 70), (3, 16, 5000), (1, 15, 20000)])
def test_linear8(kind, r, n, m):
    rng = np.random.default_rng(r * 31 + n)
    x, (w, ws) = activations(rng, r, n, kind), weights(rng, m, n)
    bias = rng.standard_normal(m).astype(np.float32) if m % 2 else None
    qx, xs = O8.quantise(x) if r * n < 200000 else (None, None)
    cw, cws, cb = cuda(w)[:, :n], cuda(ws), None if bias is None else cuda(bias)
    y = torch.full((r, m + 3), 7.0, dtype=TT[kind], device="cuda")
    Dc.linear8_noalloc(cuda(x), cw, cws, y[:, :m], bias=cb, workspace=work(Dc.linear8_workspace(r, n)), stream=stream())
    if qx is None:  # (the rounding has its own tests: here the device's)
        q, s = torch.empty(r, n, dtype=torch.int8, device="cuda"), torch.empty(r, device="cuda")
        Dc.quantise_rows_noalloc(cuda(x), q, s, stream=stream())
        qx, xs = q.cpu().numpy(), s.cpu().numpy()
    want = O8.mul_mat8(qx, xs, w[:, :n], ws, bias, NP[kind])
    assert y[:, :m].cpu().numpy().tobytes() == want.tobytes()
    assert bool((y[:, m:] == 7.0).all())
    # the same from rows that are rounded already, into the other type
    other = "f32" if kind == "f16" else "f16"
    pad = torch.full((r, w.shape[1] + 16), 99, dtype=torch.int8, device="cuda")
    pad[:, :n] = cuda(qx)
    y = torch.empty((r, m), dtype=TT[other], device="cuda")
    Dc.mul_mat8_noalloc(pad[:, :n], cuda(xs), cw, cws, y, bias=cb, stream=stream())
    assert y.cpu().numpy().tobytes() == O8.mul_mat8(qx, xs, w[:, :n], ws, bias, NP[other]).tobytes()


def test_linear8_extremes():
    """Sums at the ends of 32 bits; a row that is not finite is NaN and leaves the others alone."""
    n, m = 131071, 130
    for r in (1, 3, 20, 140):
        x, w = np.full((r, 131072), -128, np.int8), np.full((m, 131072), -128, np.int8)
        w[1] = 127
        xs, ws = np.ones(r, np.float32), np.ones(m, np.float32)
        y = torch.empty(r, m, device="cuda")
        Dc.mul_mat8_noalloc(cuda(x)[:, :n], cuda(xs), cuda(w)[:, :n], cuda(ws), y, stream=stream())
        assert y.cpu().numpy().tobytes() == O8.mul_mat8(x[:, :n], xs, w[:, :n], ws).tobytes()
    rng = np.random.default_rng(0)
    x = rng.standard_normal((20, 64)).astype(np.float32)
    x[3, 5], x[9, 0] = np.nan, np.inf
    w, ws = weights(rng, 70, 64)
    y = torch.empty(20, 70, device="cuda")
    Dc.linear8_noalloc(cuda(x), cuda(w), cuda(ws), y, workspace=work(Dc.linear8_workspace(20, 64)), stream=stream())
    assert bool(y[[3, 9]].isnan().all()) and not bool(y[[i for i in range(20) if i not in (3, 9)]].isnan().any())


def test_linear8_no_rows_and_refusals():
    w, s = torch.zeros(64, 48, dtype=torch.int8, device="cuda"), torch.ones(64, device="cuda")
    ws = work(Dc.linear8_workspace(4, 48))
    Dc.linear8_noalloc(torch.empty(0, 48, device="cuda"), w, s, torch.empty(0, 64, device="cuda"), workspace=ws)
    x, y = torch.ones(4, 48, device="cuda"), torch.empty(4, 64, device="cuda")
    with pytest.raises(ShloError, match="multiples of 16"):
        Dc.linear8_noalloc(x[:, :47], w[:, 1:], s, y, workspace=ws)
    odd = torch.zeros(64, 40, dtype=torch.int8, device="cuda")
    with pytest.raises(ShloError, match="multiples of 16"):
        Dc.linear8_noalloc(x[:, :40], odd, s, y, workspace=ws)
    with pytest.raises(ShloError, match="workspace"):
        Dc.linear8_noalloc(x, w, s, y, workspace=ws[:100])
    with pytest.raises(ShloError, match="workspace"):
        Dc.linear8_noalloc(x, w, s, y, workspace=None)
    with pytest.raises(ShloError, match="131071"):
        Dc.mul_mat8_noalloc(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), s[:1],
                            torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), s[:1], y[:1, :1])


def test_8_bits_results_in_operands_memory():
    """Refused; rows side by side in one buffer are not the same memory."""
    buf = torch.zeros(40, 256, dtype=torch.float16, device="cuda")
    buf[:, :64] = torch.randn(40, 64, device="cuda")
    w, s = torch.ones(64, 64, dtype=torch.int8, device="cuda"), torch.ones(64, device="cuda")
    ws = work(Dc.linear8_workspace(40, 64))
    x, y = buf[:, :64], torch.empty(40, 64, dtype=torch.float16, device="cuda")
    Dc.linear8_noalloc(x, w, s, buf[:, 64:128], workspace=ws, stream=stream())
    Dc.linear8_noalloc(x, w, s, y, workspace=ws, stream=stream())
    assert torch.equal(buf[:, 64:128], y)
    bits = buf.view(torch.int8)
    for out in (x, buf[:, 32:96], buf[1:, :64], bits[:, :128].view(torch.float16)):
        with pytest.raises(ShloError, match="shares memory"):
            Dc.linear8_noalloc(x[:out.shape[0]], w, s, out, workspace=work(Dc.linear8_workspace(40, 64)))
    for rows in (1, 4):
        with pytest.raises(ShloError, match="shares memory"):
            Dc.linear8_noalloc(x[:rows], w, s, x[:rows], workspace=ws)
    with pytest.raises(ShloError, match="shares memory"):
        Dc.linear8_noalloc(x, w[:16], s[:16], ws[:2560].view(torch.float16).view(40, 32)[:, :16], workspace=ws)
    with pytest.raises(ShloError, match="shares memory"):
        Dc.mul_mat8_noalloc(w[32:], s[:32], w[:16], s[:16], w.view(torch.float16)[:32, :16])
    q, scale = torch.empty(40, 64, dtype=torch.int8, device="cuda"), torch.empty(40, device="cuda")
    Dc.quantise_rows_noalloc(x, bits[:, 256:320], scale, stream=stream())
    Dc.quantise_rows_noalloc(x, q, scale, stream=stream())
    assert torch.equal(bits[:, 256:320], q)
    with pytest.raises(ShloError, match="share memory"):
        Dc.quantise_rows_noalloc(x, bits[:, 64:128], scale)
    with pytest.raises(ShloError, match="share memory"):
        Dc.quantise_rows_noalloc(x, q, q.view(-1).view(torch.float32)[:40])


# ------------------------------------------------------------ beam_select ----

def select(z, scores, keep, kind, ended=None, end=-1, view=None):
    seqs, beams = scores.shape
    next_ = torch.full((seqs, keep), 9.0, device="cuda")
    p, t = (torch.full((seqs, keep), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    w = work(Dc.beam_workspace(seqs, beams, keep, z.shape[1])).fill_(255)
    logits = cuda(z) if view is None else view(cuda(z))
    Dc.beam_select_noalloc(logits, cuda(scores), next_, p, t, ended=None if ended is None else cuda(ended), end_token=end,
                           workspace=w, stream=stream())
    return next_.cpu().numpy(), p.cpu().numpy(), t.cpu().numpy()


def same(got, want):
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    none = want[1] < 0
    assert np.all(got[0][none] == -np.inf)
    w = want[0][~none]
    assert np.all(np.abs(got[0][~none] - w) <= 2.0 ** -23 + 2.0 ** -24 * np.abs(w))


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("seqs,beams,keep,v", [(1, 1, 1, 1), (1, 1, 5, 3), (1, 4, 4, 32001), (3, 2, 4, 100), (2, 8, 16, 5000), (5, 3, 3, 1023),
                                               (1, 64, 64, 300), (2, 32, 64, 9001), (40, 8, 8, 20000), (1, 5, 10, 8192), (2, 1, 64, 70000)])
def test_beam_select(kind, seqs, beams, keep, v):
    rng = np.random.default_rng(v + beams)
    z = (rng.standard_normal((seqs * beams, v)) * rng.uniform(0.5, 3, (seqs * beams, 1))).astype(NP[kind])
    scores = (-rng.random((seqs, beams)) * 4 - 30).astype(np.float32)
    same(select(z, scores, keep, kind), O8.beam(z, scores, keep))


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_beam_select_masks_and_ends(kind):
    rng = np.random.default_rng(2)
    seqs, beams, v = 6, 5, 4001
    z = (rng.standard_normal((seqs * beams, v)) * 2).astype(NP[kind])
    z[rng.random(z.shape) < 0.9] = -np.inf
    z[0:5] = -np.inf                      # a sequence without anything
    z[5:10, 3:] = -np.inf                 # and one with few
    z[11] = -np.inf
    z[12, 700] = np.nan
    z[13, 3000] = np.inf
    z[14] = np.finfo(NP[kind]).min        # all at the type's lowest value
    scores = (-rng.random((seqs, beams)) * 4).astype(np.float32)
    scores[3, 1:] = -np.inf               # a first step: one beam counts
    scores[4, 2] = np.nan
    ended = np.zeros((seqs, beams), np.int32)
    ended[4, 0] = ended[5, 4] = 1
    ended[0, 2] = 5
    for keep in (5, 10, 64):
        same(select(z, scores, keep, kind, ended, 2), O8.beam(z, scores, keep, ended, 2))
    same(select(z, scores, 5, kind, np.ones_like(ended), 4), O8.beam(z, scores, 5, np.ones_like(ended), 4))


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_beam_select_ties(kind):
    """Equal logits everywhere, in many places, and equal beams: the lowest beam, then the lowest token first."""
    rng = np.random.default_rng(3)
    for v in (7, 300, 40000):
        z = np.zeros((4, v), NP[kind])
        scores = np.full((2, 2), -1.5, np.float32)
        for keep in (1, 6, 64):
            same(select(z, scores, keep, kind), O8.beam(z, scores, keep))
        row = rng.integers(-3, 3, v).astype(NP[kind])
        z[:] = row
        same(select(z, scores, 33, kind), O8.beam(z, scores, 33))
        z[:, ::2] = np.where(z[:, ::2] == 0, NP[kind](-0.0), z[:, ::2])  # -0 is 0
        same(select(z, scores, 33, kind), O8.beam(z, scores, 33))
    z = np.sort(rng.standard_normal((2, 50000)).astype(NP[kind]))  # all of the best in a few threads' hands
    for a in (z, z[:, ::-1]):
        same(select(np.ascontiguousarray(a), np.zeros((1, 2), np.float32), 64, kind), O8.beam(a, np.zeros((1, 2)), 64))
    a = np.full((1, 9000), -5, NP[kind])
    a[0, 4096:4096 + 64] = 1 + np.arange(64) / 64
    same(select(a, np.zeros((1, 1), np.float32), 64, kind), O8.beam(a, np.zeros((1, 1)), 64))


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_beam_select_long_rows(kind):
    """Rows that a block goes over in several turns: rising ones (each turn's candidates are more than there is room
    for), ones whose beginning is masked or far below what follows, falling ones, flat ones."""
    rng = np.random.default_rng(9)
    seqs, beams, v = 64, 8, 41003
    z = rng.standard_normal((seqs * beams, v)).astype(NP[kind])
    z[:64] = np.sort(z[:64], axis=1)
    z[64:128, :30000] = -np.inf
    z[128:192, :9000] -= 200
    z[192:200] = z[192:200, ::-1]
    z[200:208, :] = 1
    z[208:216, 20000:] += 90
    z[216:224, ::2] = -np.inf
    scores = -rng.random((seqs, beams)).astype(np.float32)
    for keep in (8, 64):
        same(select(z, scores, keep, kind), O8.beam(z, scores, keep))


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_beam_select_strides(kind):
    """Rows at any distance and offset: vectors of 16 bytes begin inside of them."""
    rng = np.random.default_rng(4)
    for v, off, pad in ((1000, 1, 7), (4099, 3, 0), (2048, 8, 8), (50, 5, 1), (3, 2, 2)):
        wide = np.full((6, off + v + pad), 60000.0, NP[kind])  # (what lies around a row is not part of it)
        wide[:, off:off + v] = rng.standard_normal((6, v))
        scores = -rng.random((2, 3)).astype(np.float32)
        got = select(wide[:, :v], scores, 6, kind, view=lambda _: cuda(wide)[:, off:off + v])
        same(got, O8.beam(wide[:, off:off + v], scores, 6))


def test_beam_select_logarithm():
    """A score that the logarithm cancels: what is left is its error, 2^-23 at most."""
    rng = np.random.default_rng(6)
    for v in (10, 3000, 128256):
        for width in (0.01, 1.0, 4.0, 30.0):
            z = (rng.standard_normal((1, v)) * width + 3).astype(np.float32)
            l = z[0].astype(np.float64)
            lse = l.max() + np.log(np.exp(l - l.max()).sum())
            score = np.array([[lse - l.max()]], np.float32)
            got = select(z, score, 1, "f32")
            assert abs(float(got[0][0, 0]) - (float(score[0, 0]) + l.max() - lse)) <= 2.0 ** -23
    z = np.array([[1e30, 1e30, -1e30, 9e29]], np.float32)  # far from everything
    same(select(z, np.zeros((1, 1), np.float32), 2, "f32"), (np.array([[-np.log(2.0)] * 2]), np.zeros((1, 2), np.int32), np.array([[0, 1]])))


def test_beam_select_refusals():
    z, s = torch.zeros(4, 10, device="cuda"), torch.zeros(2, 2, device="cuda")
    p, t = (torch.zeros(2, 2, dtype=torch.int32, device="cuda") for _ in range(2))
    w = work(Dc.beam_workspace(2, 2, 2, 10))
    Dc.beam_select_noalloc(z, s, torch.empty_like(s), p, t, workspace=w)
    for bad in (dict(workspace=None), dict(workspace=w[:8]), dict(workspace=w[1:])):
        with pytest.raises(ShloError, match="workspace"):
            Dc.beam_select_noalloc(z, s, torch.empty_like(s), p, t, **bad)
    with pytest.raises(ShloError, match="rows of logits"):
        Dc.beam_select_noalloc(z[:3], s, torch.empty_like(s), p, t, workspace=w)
    with pytest.raises(ShloError, match="kept"):
        Dc.beam_select_noalloc(z, s, torch.empty(2, 65, device="cuda"), torch.zeros(2, 65, dtype=torch.int32, device="cuda"),
                               torch.zeros(2, 65, dtype=torch.int32, device="cuda"), workspace=w)


def test_beam_select_in_place_and_shared_results():
    rng = np.random.default_rng(12)
    z, scores = rng.standard_normal((6, 300)).astype(np.float32), rng.standard_normal((2, 3)).astype(np.float32)
    w = work(Dc.beam_workspace(2, 3, 4, 300))
    i32 = lambda n: torch.zeros(2, n, dtype=torch.int32, device="cuda")  # noqa: E731
    zz, s, p, t = cuda(z), cuda(scores), i32(3), i32(3)
    Dc.beam_select_noalloc(zz, s, s, p, t, workspace=w, stream=stream())
    same((s.cpu().numpy(), p.cpu().numpy(), t.cpu().numpy()), O8.beam(z, scores, 3))
    buf = torch.zeros(64, device="cuda")
    ints = buf.view(torch.int32)
    a, b = buf[:6].view(2, 3), ints[:8].view(2, 4)
    four = torch.zeros(2, 4, device="cuda")
    for args in ((zz, a, buf[2:10].view(2, 4), i32(4), i32(4)), (zz, a, four, b, i32(4)), (zz, a, four, i32(4), b),
                 (zz, a, torch.zeros(2, 3, device="cuda"), ints[:6].view(2, 3), i32(3)), (zz, a, buf[16:24].view(2, 4), ints[20:28].view(2, 4), i32(4)),
                 (zz, a, four, ints[20:28].view(2, 4), ints[27:35].view(2, 4)), (zz, a, zz.view(-1)[-8:].view(2, 4), i32(4), i32(4))):
        with pytest.raises(ShloError, match="share"):
            Dc.beam_select_noalloc(*args, workspace=w)
    with pytest.raises(ShloError, match="share"):
        Dc.beam_select_noalloc(zz, cuda(scores), torch.zeros(2, 3, device="cuda"), p, t, ended=p, workspace=w)


# ------------------------------------------------------------------- fork ----

@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("page,heads,dim", [(16, 1, 16), (64, 3, 80), (256, 2, 256), (32, 8, 128)])
def test_fork(layout, page, heads, dim):
    rng = np.random.default_rng(page + dim)
    rows, width = 9, 5
    lens = np.array([0, 1, page, page + 3, 3 * page - 1, 2 * page, 5 * page, 5 * page + 7, -4], np.int32)
    parents = np.array([3, 3, 4, 4, 4, 2, 2, 7, 7, -1, 9, 0, 1, 1, 1, 8, 6, 5, 3], np.int32)
    pages = rows * width + 3
    cache = O.Cache(pages + len(parents), heads, page, dim)
    tables = rng.permutation(rows * width).reshape(rows, width).astype(np.int32)
    tables[4, 0], tables[1, 0] = -1, pages + 1000
    fresh = (pages + np.arange(len(parents))).astype(np.int32)
    fresh[18] = -1
    k, v = cuda(cache.k), cuda(cache.v)
    if layout == "tokens":
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    ks, vs = cuda(cache.ks), cuda(cache.vs)
    out, news = torch.full((len(parents), width + 2), 5, dtype=torch.int32, device="cuda"), torch.full((len(parents),), 5, dtype=torch.int32, device="cuda")
    for _ in range(2):  # a call repeated changes nothing
        Dc.fork_noalloc(Dc.Pool(k, v, ks, vs), cuda(tables), cuda(lens), cuda(parents), cuda(fresh), out[:, :width], news, stream=stream())
    want, wl = O8.fork(cache, tables, lens, parents, fresh)
    assert np.array_equal(out[:, :width].cpu().numpy(), want) and np.array_equal(news.cpu().numpy(), wl)
    assert bool((out[:, width:] == 5).all())
    for got, w in ((k, cache.k), (v, cache.v), (ks, cache.ks), (vs, cache.vs)):
        assert np.array_equal(got.cpu().numpy(), w)


def test_fork_refusals_and_no_rows():
    pool = Dc.Pool(*[torch.zeros(4, 2, 16, 16, dtype=torch.int8, device="cuda") for _ in range(2)],
                   *[torch.zeros(4, 2, device="cuda") for _ in range(2)])
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    Dc.fork_noalloc(pool, i32(3, 2), i32(3), i32(0), i32(0), i32(0, 2), i32(0))
    t, l = i32(3, 2), i32(3)
    with pytest.raises(ShloError, match="old ones"):
        Dc.fork_noalloc(pool, t, l, i32(3), i32(3), t, i32(3))
    with pytest.raises(ShloError, match="kv_fork"):
        Dc.fork_noalloc(pool, t, l, i32(3), i32(2), i32(3, 2), i32(3))
    with pytest.raises(ShloError, match="kv_fork"):
        Dc.fork_noalloc(pool, t, l, i32(3), i32(3), i32(3, 3), i32(3))


def test_fork_into_what_it_reads():
    pool = Dc.Pool(*[torch.zeros(4, 2, 16, 16, dtype=torch.int8, device="cuda") for _ in range(2)],
                   *[torch.zeros(4, 2, device="cuda") for _ in range(2)])
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    two = i32(3, 2, 2)  # tables and those to come, row by row side by side
    two[:, 0] = torch.arange(6, device="cuda").view(3, 2) % 4
    lens, parents = i32(3) + 32, torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda")
    out = i32(3)
    Dc.fork_noalloc(pool, two[:, 0], lens, parents, i32(3), two[:, 1], out, stream=stream())
    assert two[:, 1].tolist() == [[0, 1], [-1, -1], [0, 1]] and out.tolist() == [32, 0, 32]
    t = i32(5, 2)
    for args in ((t[:3], lens, parents, i32(3), t[2:], out), (t[:3], lens, parents, i32(3), i32(3, 2), lens),
                 (t[:3], lens, parents, i32(3), i32(3, 2), parents), (t[:3], lens, parents, out, i32(3, 2), out),
                 (t[:3], lens, parents, i32(3), t.view(-1)[3:9].view(3, 2), out), (i32(3, 2), lens, parents, i32(3), t[:3], t.view(-1)[4:7])):
        with pytest.raises(ShloError, match="memory"):
            Dc.fork_noalloc(pool, *args)


# --------------------------------------------------------------- together ----

class Step:
    """A decoder layer's step with beams, as a serving program runs it: projections in 8 bits, norm and rotation, the
    cache, attention, the output over the vocabulary, selection, forks."""

    def __init__(self, seed, seqs=2, beams=3, d=96, hq=4, hk=2, dim=32, vocab=777, page=16, length=21):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.seqs, self.beams, self.hq, self.hk, self.dim, rows = seqs, beams, hq, hk, dim, seqs * beams
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        self.w = {}
        for name, m, n in (("qkv", (hq + 2 * hk) * dim, d), ("o", d, hq * dim), ("head", vocab, d)):
            pad = -(-n // 16) * 16
            q, s = torch.zeros(m, pad, dtype=torch.int8, device="cuda")[:, :n], torch.empty(m, device="cuda")
            Dc.quantise_rows_noalloc(rn(m, n) * n ** -0.5, q, s, stream=stream())
            self.w[name] = q, s
        self.wq, self.wk = 1 + 0.1 * rn(dim), 1 + 0.1 * rn(dim)
        self.phases = cuda(Dc.rope_phases(dim)[0])
        pages = rows * 4 + rows
        shape = (pages, hk, page, dim)
        self.pool = Dc.Pool(*[torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g) for _ in range(2)],
                            *[torch.rand(pages, hk, device="cuda", generator=g) * 0.02 + 0.01 for _ in range(2)])
        self.tables = torch.arange(rows * 4, dtype=torch.int32, device="cuda").view(rows, 4)
        self.fresh = torch.arange(rows * 4, pages, dtype=torch.int32, device="cuda")
        self.lens, self.starts = i32([length] * rows), torch.arange(rows + 1, dtype=torch.int32, device="cuda")
        self.pos = i32([length - 1] * rows)
        self.x, self.scores = rn(rows, d), -torch.rand(seqs, beams, device="cuda", generator=g)
        self.space = [work(Dc.linear8_workspace(rows, max(d, hq * dim))), torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda"),
                      work(Dc.beam_workspace(seqs, beams, beams, vocab))]
        self.qkv, self.qk = torch.empty(rows, (hq + 2 * hk) * dim, device="cuda"), torch.empty(rows, hq + hk, dim, device="cuda")
        self.att, self.h, self.z = torch.empty(rows, hq, dim, device="cuda"), torch.empty(rows, d, device="cuda"), torch.empty(rows, vocab, device="cuda")
        self.next, self.parents, self.tokens = torch.empty(seqs, beams, device="cuda"), i32([[0] * beams] * seqs), i32([[0] * beams] * seqs)
        self.tables2, self.lens2 = torch.empty_like(self.tables), torch.empty_like(self.lens)

    def run(self):
        st, rows = stream(), self.x.shape[0]
        Dc.linear8_noalloc(self.x, *self.w["qkv"], self.qkv, workspace=self.space[0], stream=st)
        heads = self.qkv.view(rows, self.hq + 2 * self.hk, self.dim)
        both = self.hq + self.hk
        Dc.norm_rope_noalloc(heads[:, :both], self.pos, self.phases, self.qk, q_heads=self.hq, q_weight=self.wq, k_weight=self.wk, eps=1e-6, stream=st)
        Dc.append_noalloc(self.pool, self.qk[:, self.hq:], heads[:, both:], self.starts, self.lens, self.tables, stream=st)
        Dc.attend_noalloc(self.pool, self.qk[:, :self.hq], self.starts, self.lens, self.tables, self.att, workspace=self.space[1], scale=self.dim ** -0.5, stream=st)
        Dc.linear8_noalloc(self.att.view(rows, -1), *self.w["o"], self.h, workspace=self.space[0], stream=st)
        Dc.linear8_noalloc(self.h, *self.w["head"], self.z, workspace=self.space[0], stream=st)
        Dc.beam_select_noalloc(self.z, self.scores, self.next, self.parents, self.tokens, workspace=self.space[2], stream=st)
        Dc.fork_noalloc(self.pool, self.tables, self.lens, self.parents, self.fresh, self.tables2, self.lens2, stream=st)

    def result(self):
        return [a.cpu().numpy().copy() for a in (self.qk, self.att, self.z, self.next, self.parents, self.tokens, self.tables2, self.lens2, *self.pool.keep)]


def plain_step(s):
    """The same by the oracles, from the device's inputs; each product from the device's own operands, so that a
    rounding to 8 bits that falls the other way does not spread."""
    rows, both = s.x.shape[0], s.hq + s.hk
    cache = O.Cache(s.pool.c.pages, s.hk, s.pool.c.page_tokens, s.dim)
    cache.k, cache.v, cache.ks, cache.vs = (a.cpu().numpy().copy() for a in s.pool.keep)

    def product(x, name):
        q, sc = O8.quantise(x)
        return O8.mul_mat8(q, sc, s.w[name][0].cpu().numpy(), s.w[name][1].cpu().numpy())
    qkv = product(s.x.cpu().numpy(), "qkv")
    lens, tables = s.lens.cpu().numpy(), s.tables.cpu().numpy()
    yield qkv
    heads = qkv.reshape(rows, both + s.hk, s.dim)
    qk, mag = O8.norm_rope(heads[:, :both], s.pos.cpu().numpy(), 10000.0 ** (-2.0 * np.arange(s.dim // 2) / s.dim), s.wq.cpu().numpy(), s.wk.cpu().numpy(),
                           s.hq, np.float64(np.float32(1e-6)))
    yield qk, 2.0 ** -19 * mag
    dev = s.qk.cpu().numpy()
    O.append(cache, dev[:, s.hq:], heads[:, both:], s.starts.cpu().numpy(), lens, tables)
    att, _, _, vmax = O.attend(cache, dev[:, :s.hq], s.starts.cpu().numpy(), lens, tables, s.dim ** -0.5)
    yield att, 2.0 ** -15 * vmax[..., None]
    h = product(s.att.cpu().numpy().reshape(rows, -1), "o")
    yield product(h, "head")
    yield O8.beam(s.z.cpu().numpy(), s.scores.cpu().numpy(), s.beams)
    parents = s.parents.cpu().numpy().reshape(-1)
    yield (*O8.fork(cache, tables, lens, parents, s.fresh.cpu().numpy()), cache)


def test_a_step_of_all_together():
    s = Step(1)
    want = plain_step(s)
    qkv = next(want)
    s.run()
    assert s.qkv.cpu().numpy().tobytes() == qkv.tobytes()
    for got in (s.qk, s.att):
        w, tol = next(want)
        assert np.all(np.abs(got.cpu().numpy() - w) <= tol)
    assert s.z.cpu().numpy().tobytes() == next(want).tobytes()
    same([a.cpu().numpy() for a in (s.next, s.parents, s.tokens)], next(want))
    tables, lens, cache = next(want)
    assert np.array_equal(s.tables2.cpu().numpy(), tables) and np.array_equal(s.lens2.cpu().numpy(), lens)
    for got, w in zip(s.pool.keep, (cache.k, cache.v, cache.ks, cache.vs)):
        assert np.array_equal(got.cpu().numpy(), w)


def test_a_step_captured_and_two_at_once():
    """Captured and replayed with other inputs, and two of them on streams of their own at the same time, each with its
    own workspaces: the bits of one after the other."""
    steps, fresh = [Step(2, vocab=5001), Step(3, seqs=5, length=37)], []
    for s in steps:
        kept = [a.clone() for a in s.pool.keep]
        s.run()
        fresh.append(s.result())
        for a, b in zip(s.pool.keep, kept):
            a.copy_(b)
        s.kept = kept
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    graphs = []
    for s, st in zip(steps, streams):
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                s.run()
            graphs.append(g)
    for turn in range(3):
        for s, st, g in zip(steps, streams, graphs):
            with torch.cuda.stream(st):
                for a, b in zip(s.pool.keep, s.kept):
                    a.copy_(b)
                g.replay()
        torch.cuda.synchronize()
        for s, want in zip(steps, fresh):
            assert all(a.tobytes() == b.tobytes() for a, b in zip(s.result(), want))
    other = Step(4)  # a captured call reads what lies in its operands when it is replayed
    steps[0].x.copy_(other.x)
    for a, b in zip(steps[0].pool.keep, steps[0].kept):
        a.copy_(b)
    with torch.cuda.stream(streams[0]):
        graphs[0].replay()
    torch.cuda.synchronize()
    got = steps[0].result()
    for a, b in zip(steps[0].pool.keep, steps[0].kept):
        a.copy_(b)
    steps[0].run()
    assert all(a.tobytes() == b.tobytes() for a, b in zip(got, steps[0].result()))
    del graphs


def test_host_threads_at_once():
    import threading
    steps, want, errors = [Step(5), Step(6, seqs=4)], [], []
    for s in steps:
        s.run()
        want.append(s.result()[:6])
    torch.cuda.synchronize()

    def go(s, w):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    s.run()
                st.synchronize()
            # (the cache's tail pages take the same tokens again, which changes nothing)
            if not all(a.tobytes() == b.tobytes() for a, b in zip(s.result()[:6], w)):
                errors.append("bits")
        except Exception as e:  # noqa: BLE001
            errors.append(repr(e))
    threads = [threading.Thread(target=go, args=a) for a in zip(steps, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert errors == []
