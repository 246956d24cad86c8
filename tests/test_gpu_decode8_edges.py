"""The norm with rotation, the products in 8 bits, beam search's selection and the cache's reordering on the GPU where
values, masks or memory are unusual; the tolerances of tests/test_gpu_decode8.py, whose helpers these use, unless a test
says otherwise."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import decode8_oracle as O8  # noqa: E402
from shlo import decode as Dc  # noqa: E402
from shlo import mlx as M  # noqa: E402
from test_gpu_decode8 import NP, TT, cuda, same, select, stream, work  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.set_device(0)
    M.set_device(0)
    yield
    torch.cuda.empty_cache()


# -------------------------------------------------------------- norm_rope ----

@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("q_heads", [0, 8])
def test_norm_rope_grad_of_many_tokens_of_one_kind(kind, q_heads):
    """Queries alone, keys alone: a thread's terms of one weight's gradient are as many as 900 in a row, of one sign and
    here all the same, so that what an addition loses, it loses each time. What is summed in binary32 are 16 heads: 2^-20 of
    the sum of magnitudes, as much again the norm (16 + 5 roundings, 2^-24 each, and the root's), and the result's own
    rounding: 2^-18, however many tokens."""
    T, H, D = 400000, 8, 512
    rng = np.random.default_rng(q_heads + 5)
    x, dy = rng.uniform(0.5, 2, (2, 1, 1, D)).astype(NP[kind])
    w = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    pos, phases = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    dx, dw = torch.empty(T, H, D, dtype=TT[kind], device="cuda"), torch.full((2, D), np.nan, device="cuda")
    Dc.norm_rope_grad_noalloc(cuda(x).expand(T, H, D), cuda(dy).expand(T, H, D), pos, phases, dx, dw[0], dw[1], q_heads=q_heads,
                              q_weight=cuda(w), k_weight=cuda(w), eps=1e-5, workspace=work(Dc.norm_rope_workspace()), stream=stream())
    n = x.astype(np.float64) / np.sqrt((x.astype(np.float64) ** 2).mean() + np.float64(np.float32(1e-5)))
    want = T * H * (n * dy.astype(np.float64))[0, 0]
    got = dw.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got[0 if q_heads else 1] - want) <= 2.0 ** -18 * want)
    assert np.all(got[1 if q_heads else 0] == 0)


# ------------------------------------------------------------ beam_select ----

def not_numbers(z, rows, lo, hi, rng):
    """NaNs of both signs in columns lo to hi, of the rows' type."""
    nan = np.copysign(np.nan, rng.choice([-1.0, 1.0, 1.0], (len(rows), hi - lo)))
    z[rows, lo:hi] = nan.astype(z.dtype)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("seqs,beams,v", [(1, 4, 8192), (64, 8, 41003), (1, 2, 3000), (2, 3, 131072)])
def test_beam_select_of_many_nans_beside_equal_logits(kind, seqs, beams, v):
    """More equal logits than a block has room for, and more NaNs: at the beginning, in later stretches, everywhere,
    in every other place. Their rows give nothing, the others what they gave."""
    rng = np.random.default_rng(v)
    z = rng.standard_normal((seqs * beams, v)).astype(NP[kind])
    odd = np.arange(0, seqs * beams, 2)
    for i, r in enumerate(odd):
        r = np.array([r])
        z[r] = [0, -3, 5][i % 3]
        where = [(0, v // 2), (v // 2, v), (v // 4, v // 4 + 600), (0, v), (v - 700, v)][i % 5]
        if i % 7 == 6:
            z[r, ::2] = np.nan
        else:
            not_numbers(z, r, *where, rng)
        if i % 11 == 10:
            z[r, :v // 3] = np.inf
    z[1] = 2.0
    scores = -rng.random((seqs, beams)).astype(np.float32)
    for keep in (1, 8, 64):
        same(select(z, scores, keep, kind), O8.beam(z, scores, keep))


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("seqs,beams,v,left", [(8, 8, 5000, 3), (40, 16, 5000, 20), (20, 40, 8000, 60), (64, 8, 41003, 33)])
def test_beam_select_equal_rows_with_few_logits_left(kind, seqs, beams, v, left):
    """Rows of which a mask leaves fewer than are kept, the same for all beams of a sequence: their sums are the same bits,
    so that the lowest beam comes first, and two calls give the same. (Terms far below the largest: sums of a few near ones
    are exact in 64 bits, in any order.)"""
    rng = np.random.default_rng(left)
    z = np.full((seqs, 1, v), -np.inf, NP[kind])
    for s in range(seqs):
        z[s, 0, rng.choice(v, left, replace=False)] = -45 * rng.random(left)
    z = np.repeat(z, beams, 1).reshape(seqs * beams, v)
    scores = np.repeat(-rng.random((seqs, 1)).astype(np.float32), beams, 1)
    want = O8.beam(z, scores, 64)
    first = select(z, scores, 64, kind)
    same(first, want)
    for _ in range(50):
        assert all(np.array_equal(a, b) for a, b in zip(select(z, scores, 64, kind), first))


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("rise", [3, 10, 30, 57.22, 59.9])
def test_beam_select_rows_that_rise(kind, rise):
    """Rows that a block goes over in several turns, which rise above the first: plateaus of equal logits, more than are
    kept, that begin in a later turn; the same in steps; single logits and noise up there. The scores cancel the
    logarithm, so that its error is what is left: 2^-23."""
    rng = np.random.default_rng(int(rise))
    seqs, v = 512, 41003
    z = (rng.standard_normal((seqs, v)) * 0.3).astype(NP[kind])
    z[0::4, 20000:] = rise
    z[1::4, 9000:] = rise / 3
    z[1::4, 18000:] = rise
    z[2::4, 20000:] += NP[kind](rise)
    z[3::4, 30001] = rise
    z[4::8, 2000:2003] = rise  # (in the first turn too: what follows is no higher)
    z[5::8, :17000] = -np.inf
    l = z.astype(np.float64)
    top = l.max(1, keepdims=True)
    lse = top[:, 0] + np.log(np.exp(l - top).sum(1))
    scores = (lse - top[:, 0]).astype(np.float32)[:, None]
    want = O8.beam(z, scores, 64)
    # A plateau no more than 2 above the first turn's largest is counted from that: a term is then off by 2.06 10^-7 at
    # most (ex2.approx and the roundings of its argument, over all arguments up to 2; 2^-22 is 2.38 10^-7), and equal
    # terms add up without rounding, so the logarithm is off by 2^-22 at most.
    first = l[:, :8192].max(1)
    near = (top[:, 0] > first) & (top[:, 0] <= first + 2.1)
    for keep in (1, 8, 64):
        got, w = select(z, scores, keep, kind), [a[:, :keep] for a in want]
        same([a[~near] for a in got], [a[~near] for a in w])
        assert all(np.array_equal(a[near], b[near]) for a, b in zip(got[1:], w[1:]))
        assert np.all(np.abs(got[0][near] - w[0][near]) <= 2.0 ** -22 + 2.0 ** -24 * np.abs(w[0][near]))
