"""The decoder operators on the GPU where a batch or its addresses are unusual; the tolerances of
tests/test_gpu_decode.py, whose cases these use."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import decode_oracle as O  # noqa: E402
from shlo import decode as Dc  # noqa: E402
from shlo import mlx as M  # noqa: E402
from shlo import run as Run  # noqa: E402
from shlo._lib import ShloError, load  # noqa: E402
from test_gpu_decode import Case, cuda, rope_close  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.set_device(0)
    M.set_device(0)
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("hk,group,lens,news", [
    (3, 4, [500, 200], [1, 2]), (2, 1, [300, 40, 7], [1, 0, 3]), (3, 4, [260, 700], [150, 90]), (1, 8, [900], [1])])
def test_rows_before_the_first_sequence(kind, hk, group, lens, news):
    """starts[0] above 0: the first rows of q are no sequence's. Every head's results are right, those rows stay, and
    the counters end at zero."""
    c = Case(kind, 16, hk, group, 64, lens, news)
    for lead in (1, 30, 77):
        q = cuda(np.concatenate([np.repeat(c.q[:1], lead, 0), c.q]))
        out = torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda")
        work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
        own = c.starts
        c.starts = (own + lead).astype(np.int32)
        got = c.run(q=q, out=out, work=work)
        c.starts = own
        c.check((got[0][lead:], got[1][lead:]))
        assert np.all(got[0][:lead] == 9.0) and np.all(got[1][:lead] == 9.0)
        assert int(work[:8192].to(torch.int32).sum()) == 0


def wait():
    """The library's own wait for its device, which tells what its launches reported."""
    torch.cuda.synchronize()
    M.to_numpy(M.transpose(M.of_numpy(np.zeros((2, 3), np.float32)), [1, 0]))


@pytest.mark.parametrize("hk,group,D,lens,news", [(2, 3, 128, [400, 129, 1000, 5], [300, 129, 1, 5]),
                                                  (1, 8, 64, [3000], [20]), (1, 5, 256, [500, 64], [200, 64])])
def test_a_launch_that_gives_up_leaves_the_next_one_right(hk, group, D, lens, news):
    """Waits that are given up: the launch returns, the error is told, and without the workspace being touched the
    next call gives the bits that it gave before."""
    c = Case("f16", 16, hk, group, D, lens, news, seed=7)
    work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    first = c.run(work=work)
    c.check(first)
    lib = load()
    try:
        for every in (1, 2, 3):  # of the blocks, so that some units' parts arrive and others' do not
            lib.shlo_test_attend_give_up(every)
            c.run(work=work)
            lib.shlo_test_attend_give_up(0)
            with pytest.raises(ShloError, match="gave up"):
                wait()
            assert int(work[:8192].to(torch.int32).sum()) == 0
            again = c.run(work=work)
            assert again[0].tobytes() == first[0].tobytes() and again[1].tobytes() == first[1].tobytes()
    finally:
        lib.shlo_test_attend_give_up(0)


def test_a_cache_after_a_launch_that_gave_up():
    """The same through a handle, whose workspace is the library's own: the wait reports it, calls after it are right."""
    rng = np.random.default_rng(5)
    cache = Dc.Cache(64, 2, 64, 16)
    n = 700
    kv = M.of_numpy(rng.standard_normal((n, 2, 64)).astype(np.float16))
    q = M.of_numpy(rng.standard_normal((n, 8, 64)).astype(np.float16))
    batch = [M.of_numpy(a) for a in (np.array([0, n], np.int32), np.array([n], np.int32), np.arange(44, dtype=np.int32)[None])]
    cache.append(kv, kv, *batch)
    first = M.to_numpy(cache.attend(q, *batch, scale=0.125))
    lib = load()
    try:
        lib.shlo_test_attend_give_up(2)
        lost = cache.attend(q, *batch, scale=0.125)
        lib.shlo_test_attend_give_up(0)
        after = cache.attend(q, *batch, scale=0.125)  # queued before the error is seen
        with pytest.raises(ShloError, match="gave up"):
            M.to_numpy(lost)
        assert M.to_numpy(after).tobytes() == first.tobytes()
        assert M.to_numpy(cache.attend(q, *batch, scale=0.125)).tobytes() == first.tobytes()
    finally:
        lib.shlo_test_attend_give_up(0)


CHILD = r'''
import sys
import threading
sys.path[:0] = [%r, %r]
import numpy as np, torch
from shlo import decode as Dc
x = torch.randn(4, 2, 16, device="cuda:0")
out, pos = torch.empty_like(x), torch.zeros(4, dtype=torch.int32, device="cuda:0")
phases = torch.from_numpy(Dc.rope_phases(16)[0]).cuda()
Dc.rope_noalloc(x, pos, phases, out)
torch.cuda.synchronize()
assert Dc.load().shlo_cuda_device() == torch.cuda.current_device() == 0
print("RESULT", bool(torch.equal(x, out)), Dc.attend_workspace() > 0)
'''


def test_the_callers_device_is_cudas():
    """The entry points on caller-owned memory work on the device that is current in CUDA, whatever device the
    library's own arrays would be on (here one that the machine does not have)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, SHLO_DEVICE="63")
    r = subprocess.run([sys.executable, "-c", CHILD % (root, os.path.join(root, "contract-stablehlo-mlx_b200"))],
                       capture_output=True, text=True, timeout=200, env=env)
    assert "RESULT True True" in r.stdout, r.stdout + r.stderr


def test_a_launch_that_gave_up_is_told_by_the_next_call():
    """Without the library's wait: the next call says so and does nothing, the one after it is right."""
    c = Case("f16", 16, 1, 8, 64, [3000], [20])
    work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    first = c.run(work=work)
    lib = load()
    try:
        lib.shlo_test_attend_give_up(1)
        c.run(work=work)
    finally:
        lib.shlo_test_attend_give_up(0)
    torch.cuda.synchronize()
    out = torch.full(c.q.shape, 9.0, dtype=torch.float16, device="cuda")
    with pytest.raises(ShloError, match="gave up"):
        c.run(work=work, out=out)
    assert bool((out == 9.0).all())
    again = c.run(work=work)
    assert again[0].tobytes() == first[0].tobytes() and again[1].tobytes() == first[1].tobytes()


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("starts", [[0, 30, 10, 60], [5, 0, 20, 40], [0, 20, 40, 39]])
def test_starts_that_descend(kind, starts):
    """Nothing is written, counters stay zero, the next call says what was wrong, and the one after it is right."""
    c = Case(kind, 16, 2, 4, 64, [500, 200, 90], [30, 20, 10])
    work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    first = c.run(work=work)
    own, c.starts = c.starts, np.array(starts, np.int32)
    out = torch.full(c.q.shape, 9.0, dtype=torch.from_numpy(c.q).dtype, device="cuda")
    c.run(work=work, out=out)
    assert bool((out == 9.0).all()) and int(work[:8192].to(torch.int32).sum()) == 0
    c.starts = own
    with pytest.raises(ShloError, match="descend"):
        c.run(work=work)
    again = c.run(work=work)
    c.check(again)
    assert again[0].tobytes() == first[0].tobytes() and again[1].tobytes() == first[1].tobytes()


def test_rope_kernel_refuses_sizes_whose_product_wraps():
    """Parameter words whose product is 2^64 plus the array's size."""
    pos, phases = M.of_numpy(np.zeros(16, np.int32)), M.of_numpy(np.zeros(1, np.int64))
    for t, h, d, n in ((16, 1 << 30, 1 << 30, 0), (5, 1 << 20, 1 << 30, 5), (16, 1 << 20, 1 << 21, 16)):
        x = M.of_numpy(np.zeros(n, np.float32))
        words = Run.params([t, h, d, 2, 0, 0x3F800000])
        p = M.of_numpy(np.zeros(t, np.int32)) if t != 16 else pos
        with pytest.raises(ShloError, match="tokens of"):
            M.kernel_apply(Run.kernel("rope"), [x, p, phases, words], [[t, h, d]], bytes([M.dtF32]), [1, 1, 1], [64, 1, 1])


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("news", [[7, 1], [90, 3]])
def test_the_widest_windows_and_rows_before_position_0(kind, news):
    """A window of 2^31 - 1 is none, for rows before position 0 too (which see every key where nothing is causal)."""
    c = Case(kind, 16, 2, 4, 64, [3, 40], news)
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 100):
        for causal in (False, True):
            got, whole = c.run(causal, window), c.run(causal, 0)
            c.check(whole, causal, 0)
            assert got[0].tobytes() == whole[0].tobytes() and got[1].tobytes() == whole[1].tobytes()


def test_rope_refuses_overlapping_storage():
    """Views of one buffer, against their values' places counted one by one: what shares a value is refused, what does
    not is right (in place too); only views of different strides inside each other's extent are refused untested."""
    rng = np.random.default_rng(11)
    buf = cuda(rng.standard_normal(700).astype(np.float32))
    keep = buf.clone()
    phases = cuda(Dc.rope_phases(4)[0])
    taken = refused = 0
    for _ in range(400):
        T, H, D = (int(n) for n in rng.integers(1, 5, 3) + [0, 0, 3])
        sh = int(rng.integers(D, 2 * D + 3)) if rng.integers(2) else int(rng.integers(T * D, T * D + 9))
        st = int(rng.integers(H * sh, H * sh + 20)) if sh < T * D or T == 1 else int(rng.integers(D, sh // T + 1))
        span = (T - 1) * st + (H - 1) * sh + D
        if span > 300:
            continue
        same = bool(rng.integers(4))
        tt, hh = (st, sh) if same else (st + int(rng.integers(3)), sh + int(rng.integers(3)))
        ox = int(rng.integers(200))
        oy = ox + int(rng.integers(-min(ox, span + 9), span + 9))
        x, y = buf.as_strided((T, H, D), (st, sh, 1), ox), buf.as_strided((T, H, D), (tt, hh, 1), oy)
        at = [{o + t * a + h * b + d for t in range(T) for h in range(H) for d in range(D)}
              for o, a, b in ((ox, st, sh), (oy, tt, hh))]
        alike = ox == oy and (st, sh) == (tt, hh)
        # the same places by other strides of axes of one
        shares = bool(at[0] & at[1]) and not alike
        inside = max(at[0]) >= min(at[1]) and max(at[1]) >= min(at[0])
        differ = (T > 1 and st != tt) or (H > 1 and sh != hh)
        buf.copy_(keep)
        pos = cuda(rng.integers(0, 99, T).astype(np.int32))
        want = torch.empty(T, H, D, device="cuda")
        Dc.rope_noalloc(x, pos, phases, want)
        if shares or (inside and differ) or (ox == oy and not alike):
            refused += 1
            with pytest.raises(ShloError, match="overlap|share storage"):
                Dc.rope_noalloc(x, pos, phases, y)
            assert torch.equal(buf, keep)
        else:
            taken += 1
            Dc.rope_noalloc(x, pos, phases, y)
            assert torch.equal(y, want)
            out = torch.ones(700, dtype=torch.bool)
            out[sorted(at[1])] = False
            assert torch.equal(buf.cpu()[out], keep.cpu()[out])
    assert taken > 50 and refused > 50


@pytest.mark.parametrize("inverse", [False, True])
def test_rope_angles_at_every_position(inverse):
    """Positions over all of int32 against turns in exact integers, position * phase mod 2^64: the tolerance of small
    positions (2^-20 of a pair's magnitude: 2^-26 turns are 2^-23.3 rad, and the sine's own error is less)."""
    rng = np.random.default_rng(12)
    T, D = 4000, 128
    edge = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 30, 2 ** 24 + 1]
    pos = np.concatenate([edge, rng.integers(-2 ** 31, 2 ** 31, T - len(edge))]).astype(np.int32)
    x = rng.standard_normal((T, 1, D)).astype(np.float32)
    phases, _ = Dc.rope_phases(D, 500000.0)
    out = torch.empty(T, 1, D, device="cuda")
    Dc.rope_noalloc(cuda(x), cuda(pos), cuda(phases), out, inverse=inverse)
    # the fraction of a turn, 53 bits of it, in [-1/2, 1/2)
    whole = pos.astype(np.int64)[:, None].view(np.uint64) * phases.view(np.uint64)[None, :]
    a = whole.view(np.int64).astype(np.float64) * 2.0 ** -63 * np.pi
    c, s = np.cos(a)[:, None], np.sin(a)[:, None] * (-1 if inverse else 1)
    lo, hi = x[..., :D // 2].astype(np.float64), x[..., D // 2:].astype(np.float64)
    want = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
    rope_close(out.cpu().numpy(), want, x, np.zeros(D // 2), 1.0, False, "f32")
    # the phases are those of the frequencies: 2^-65 turns a position each, and the 64-bit oracle's own 2^-52
    freqs = 500000.0 ** (-2.0 * np.arange(D // 2) / D)
    assert np.all(np.abs(phases.astype(np.float64) / 2.0 ** 64 * 2 * np.pi - freqs) <= 2.0 ** -48 * freqs + 2.0 ** -62)


def drift(kind, seqs, new, length, group=4, D=128, rows=4):
    """The mean signed error, relative, of the newest tokens of some sequences that share one long run of pages, whose
    values are all positive; against 64 bits, on the device."""
    g = torch.Generator(device="cuda").manual_seed(1)
    page = 256
    pages = -(-length // page)

    def ints(mean):
        return (torch.randn(pages, 1, page, D, generator=g, device="cuda") * 20 + mean).round().clamp(-127, 127).to(torch.int8)
    k, v, scale = ints(0), ints(60).abs_(), torch.full((pages, 1), 0.02, device="cuda")
    tables = torch.arange(pages, dtype=torch.int32, device="cuda").expand(seqs, pages).contiguous()
    starts, lens = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * new, torch.full((seqs,), length, dtype=torch.int32, device="cuda")
    q = torch.randn(seqs * new, group, D, generator=g, device="cuda").to(torch.float16 if kind == "f16" else torch.float32)
    out, work = torch.empty_like(q), torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    Dc.attend_noalloc(Dc.Pool(k, v, scale, scale), q, starts, lens, tables, out, scale=D ** -0.5, workspace=work)
    kk, vv = (a.reshape(-1, D)[:length].double() * scale[0, 0].double() for a in (k, v))
    errors = []
    for s in range(0, seqs, seqs // rows):
        at = s * new + new - 1
        want = (q[at].double() @ kk.T * D ** -0.5).softmax(-1) @ vv
        errors.append(((out[at].double() - want) / want).mean().item())
    return float(np.mean(errors))


@pytest.mark.parametrize("kind,bound", [("f16", 2.0 ** -13), ("f32", 2.0 ** -20)])
def test_sums_over_long_units_do_not_drift(kind, bound):
    """200 000 keys that no cut shares out among blocks (there are as many units as blocks). Errors that all point one
    way show in the mean: a matrix instruction cuts up to 2^-23 of a sum off, so 3125 of them in a row 2^-11.4. What
    may stay: the mean of 2048 results' roundings (2^-11 each, at random: 5 sigma are 2^-16; float32's 2^-24), and of
    the weights' (at random over the keys), with room for the products of one stretch of 8192 keys (2^-14). A float32
    call's weights and sums are rounded to 22 bits and more, at random: 2^-20 is several times a single rounding."""
    blocks = 3 * torch.cuda.get_device_properties(0).multi_processor_count
    assert abs(drift(kind, blocks, 1, 200000)) <= bound


def test_tiles_sums_over_long_units_do_not_drift():
    """The same bound for prompts: 64 new tokens of as many sequences as there are blocks, 12500 products a row."""
    blocks = torch.cuda.get_device_properties(0).multi_processor_count
    assert abs(drift("f16", blocks, 64, 200000)) <= 2.0 ** -13


def test_threads_on_one_cache():
    """Host threads that attend over one cache at once (and share the library's workspace): each gets its own bits."""
    rng = np.random.default_rng(6)
    n = 500
    cache = Dc.Cache(32, 2, 64, 16)
    kv = M.of_numpy(rng.standard_normal((n, 2, 64)).astype(np.float16))
    whole = [M.of_numpy(a) for a in (np.array([0, n], np.int32), np.array([n], np.int32), np.arange(32, dtype=np.int32)[None])]
    cache.append(kv, kv, *whole)
    work = []
    for t in (1, 3, 100, n):
        q = M.of_numpy(rng.standard_normal((t, 8, 64)).astype(np.float16))
        batch = [M.of_numpy(np.array([0, t], np.int32))] + whole[1:]
        work.append((q, batch, M.to_numpy(cache.attend(q, *batch, scale=0.125)).tobytes()))
    wrong = []

    def run(q, batch, want):
        M.set_device(0)
        for _ in range(40):
            if M.to_numpy(cache.attend(q, *batch, scale=0.125)).tobytes() != want:
                wrong.append(len(want))
    threads = [threading.Thread(target=run, args=w) for w in work * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("exponent", [-125, -120, -113, -60, 100])
def test_float32_values_of_every_size(exponent):
    """Value scales near the ends of binary32's normal numbers: results keep their bits, relative to the row's largest
    value (the stated bound without its absolute part)."""
    c = Case("f32", 16, 2, 4, 64, [300, 64], [1, 2], seed=5)
    c.cache.vs[:] = (np.random.default_rng(7).uniform(1, 2, c.cache.vs.shape) * 2.0 ** exponent).astype(np.float32)
    want, wl, mag, vmax = O.attend(c.cache, c.q, c.starts, c.lens, c.tables, c.scale)
    out, lse = c.run()
    tol = (2 * 2.0 ** -20 * mag + 2.0 ** -18) * vmax
    assert np.all(np.abs(out.astype(np.float64) - want) <= tol[..., None])
    # and far inside it: 22-bit weights at random, 2^-21 of the largest value
    assert np.sqrt(np.mean((out - want) ** 2)) <= 2.0 ** -21 * vmax.max()
