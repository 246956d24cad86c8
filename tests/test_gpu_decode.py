"""The decoder operators on the GPU against plain 64-bit forms (tests/decode_oracle.py).

Tolerances, from the arithmetic and before any run:
 - rope: a turn's angle is within 2^-25 of it (relative, under half a turn: 2^-23 rad), sine and cosine
   within 2^-22 then, products and sums round at 2^-24: |error| <= 2^-20 factor (|a| + |b|); a float16
   result adds its own rounding, 2^-11 |y| (and 2^-25 below its normal range).
 - append, gather: bit for bit (each step is one binary32 operation).
 - attend: a score is a sum of exact products accumulated in 32 bits (2^-20 of the sum of their magnitudes,
   for up to 256 terms), so the weights are off by d = 2^-20 max sum |q k| scale, the float16 weights of a
   float16 call by 2^-11 more, and the result by (2 d + 2^-18 + weights) max |v|, plus its own rounding;
   lse by d + 2^-20 (1 + |lse|).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import decode_oracle as O  # noqa: E402
from shlo import decode as Dc  # noqa: E402
from shlo import mlx as M  # noqa: E402
from shlo._lib import ShloError  # noqa: E402

NP = {"f16": np.float16, "f32": np.float32}


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.set_device(0)
    M.set_device(0)
    yield
    torch.cuda.empty_cache()  # the caches' gigabytes go back before other files' child processes allocate


@pytest.fixture(autouse=True)
def tidy():
    yield
    if torch.cuda.memory_reserved() > 1 << 30:
        torch.cuda.empty_cache()


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------- rope ----

def rope_close(got, want, x, freqs, factor, inter, kind):
    r = 2 * len(freqs)
    ia = np.arange(0, r, 2) if inter else np.arange(r // 2)
    ib = ia + 1 if inter else ia + r // 2
    tol = np.zeros_like(want)
    pair = factor * (np.abs(x[..., ia].astype(np.float64)) + np.abs(x[..., ib].astype(np.float64))) * 2.0 ** -20
    tol[..., ia] = pair
    tol[..., ib] = pair
    if kind == "f16":
        tol += np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    assert np.all(np.abs(got.astype(np.float64) - want) <= tol)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,D,R,top", [
    (1, 1, 2, 2, 10), (1, 40, 128, 128, 4096), (7, 3, 80, 32, 100), (33, 5, 72, 18, 1 << 20), (5, 2, 64, 64, 2 ** 31 - 1),
    (1024, 8, 64, 64, 300000), (3, 1, 200, 100, 77), (2, 2, 1030, 1030, 999), (600, 7, 96, 48, 8192), (2, 3, 66, 0, 5)])
def test_rope(kind, inter, T, H, D, R, top):
    rng = np.random.default_rng(T * 7 + D)
    x = rng.standard_normal((T, H, D)).astype(NP[kind])
    pos = rng.integers(-5, top, T, endpoint=True).astype(np.int32)
    if R:
        phases, _ = Dc.rope_phases(R, 10000.0)
        freqs = 10000.0 ** (-2.0 * np.arange(R // 2) / R)
    else:
        phases, freqs = np.zeros(0, np.int64), np.zeros(0)
    factor = 1.25
    for inverse in (False, True):
        out = torch.empty(T, H, D, dtype=torch.float16 if kind == "f16" else torch.float32, device="cuda")
        Dc.rope_noalloc(cuda(x), cuda(pos), cuda(phases), out, interleaved=inter, inverse=inverse, factor=factor,
                        stream=stream())
        want = O.rope(x, pos, freqs, factor, inter, inverse)
        # positions of 2^31 turn by 2^31 radians: the 64-bit oracle's own angle is off by 2^-22 there
        if top < 1 << 30:
            rope_close(out.cpu().numpy(), want, x, freqs, factor, inter, kind)
        else:
            assert np.max(np.abs(out.cpu().numpy().astype(np.float64) - want)) < 2.0 ** -8


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_rope_strides_in_place_and_copied_bits(kind):
    """A slice of wider rows, an odd offset that no vector load allows, in place; the copied part keeps its bits."""
    rng = np.random.default_rng(3)
    T, H, D, R = 19, 4, 64, 32
    for off in (0, 1, 2, 8):
        wide = rng.standard_normal((T, H + 2, D + 8)).astype(NP[kind])
        wide[0, 0, D - 1] = np.nan
        wide[1, 1, D - 2] = -np.inf
        pos = np.arange(T, dtype=np.int32) * 3
        phases, _ = Dc.rope_phases(R)
        freqs = 10000.0 ** (-2.0 * np.arange(R // 2) / R)
        t = cuda(wide)
        x = t[:, 1:1 + H, off:off + D] if off < 8 else t[:, 1:1 + H, 8:8 + D]
        xs = x.cpu().numpy().copy()
        out = torch.empty(T, H, D, dtype=x.dtype, device="cuda")
        Dc.rope_noalloc(x, cuda(pos), cuda(phases), out, stream=stream())
        got = out.cpu().numpy()
        rope_close(got[..., :R], O.rope(xs[..., :R], pos, freqs), xs[..., :R], freqs, 1.0, False, kind)
        assert got[..., R:].tobytes() == xs[..., R:].tobytes()
        before = t.clone()
        Dc.rope_noalloc(x, cuda(pos), cuda(phases), x, stream=stream())
        assert x.cpu().numpy().tobytes() == got.tobytes()
        x.copy_(torch.from_numpy(xs).cuda())
        assert torch.equal(t.nan_to_num(), before.nan_to_num())  # nothing around it was written


def test_rope_gradient_is_the_formulas_and_the_differences():
    """<dy, rope(x)> differentiated: the inverse call gives J^T dy; against central differences of the 64-bit form,
    which is linear in x, so a step of 1 has no truncation error."""
    rng = np.random.default_rng(4)
    T, H, D, R = 5, 2, 24, 16
    x, dy = rng.standard_normal((T, H, D)), rng.standard_normal((T, H, D)).astype(np.float32)
    pos = rng.integers(0, 5000, T).astype(np.int32)
    phases, factor = Dc.rope_phases(R, 10000.0, "ramp", 8.0, 512.0)
    for inter in (False, True):
        i = np.arange(R // 2)
        freqs = phases.astype(np.float64) / 2.0 ** 64 * 2 * np.pi
        out = torch.empty(T, H, D, device="cuda")
        Dc.rope_noalloc(cuda(dy), cuda(pos), cuda(phases), out, interleaved=inter, inverse=True, factor=factor,
                        stream=stream())
        got = out.cpu().numpy()
        rope_close(got[..., :], O.rope(dy, pos, freqs, factor, inter, True), dy, freqs, factor, inter, "f32")
        for _ in range(20):
            t, h, d = rng.integers(T), rng.integers(H), rng.integers(D)
            e = np.zeros_like(x)
            e[t, h, d] = 1.0
            diff = (dy * (O.rope(x + e, pos, freqs, factor, inter) - O.rope(x - e, pos, freqs, factor, inter))).sum() / 2
            assert abs(diff - got[t, h, d]) <= 2.0 ** -19 * factor * np.abs(dy[t, h]).max() * 2
        del i


# ---------------------------------------------------------- append, gather ----

def pool_of(cache, layout):
    def lay(a):
        t = cuda(a)
        return t if layout == "heads" else t.transpose(1, 2).contiguous().transpose(1, 2)
    return Dc.Pool(lay(cache.k), lay(cache.v), cuda(cache.ks), cuda(cache.vs))


def tables_of(lens, page, rng, spare=3, width=0):
    need = [-(-n // page) for n in lens]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    t = np.full((len(lens), max([1, width] + need)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t, sum(need) + spare


def starts_of(news):
    return np.concatenate([[0], np.cumsum(news)]).astype(np.int32)


def same_cache(pool, cache):
    k, v, ks, vs = pool.keep
    assert np.array_equal(k.cpu().numpy(), cache.k) and np.array_equal(v.cpu().numpy(), cache.v)
    assert np.array_equal(ks.cpu().numpy(), cache.ks, equal_nan=True) and np.array_equal(vs.cpu().numpy(), cache.vs, equal_nan=True)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("page,H,D,old,new", [
    (16, 1, 16, [0], [1]), (16, 8, 128, [0, 15, 16, 31, 5], [1, 1, 1, 1, 1]), (32, 3, 80, [7, 0, 64, 33], [40, 0, 1, 31]),
    (64, 2, 256, [63, 1], [2, 200]), (128, 5, 48, [100, 0, 300], [28, 129, 500]), (256, 1, 256, [3], [600])])
def test_append_and_gather(kind, layout, page, H, D, old, new):
    rng = np.random.default_rng(page + D)
    lens = [o + n for o, n in zip(old, new)]
    tables, pages = tables_of(lens, page, rng)
    cache = O.Cache(pages, H, page, D, seed=D)
    pool = pool_of(cache, layout)
    T = sum(new)
    rows = (rng.standard_normal((T, 2 * H + 1, D)) * rng.uniform(0.1, 3, (T, 1, 1))).astype(NP[kind])
    rows[:, 1] = 0 if T > 1 else rows[:, 1]  # a head of zeros: scale 0 in fresh pages
    t = cuda(rows)
    st, ln, tb = cuda(starts_of(new)), cuda(np.array(lens, np.int32)), cuda(tables)
    k, v = t[:, 1:1 + H], t[:, 1 + H:]
    O.append(cache, rows[:, 1:1 + H], rows[:, 1 + H:], starts_of(new), lens, tables)
    for _ in range(2):  # a call repeated changes nothing
        Dc.append_noalloc(pool, k, v, st, ln, tb, stream=stream())
        same_cache(pool, cache)
    seq = np.repeat(np.arange(len(lens)), lens).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    seq, pos = np.append(seq, [0, -1, len(lens), 0]).astype(np.int32), np.append(pos, [-1, 0, 0, 1 << 30]).astype(np.int32)
    gk, gv = (torch.full((len(seq), H, D), 7.0, dtype=t.dtype, device="cuda") for _ in range(2))
    Dc.gather_noalloc(pool, tb, cuda(seq), cuda(pos), gk, gv, stream=stream())
    for got, q, s in ((gk, cache.k, cache.ks), (gv, cache.v, cache.vs)):
        want = np.zeros((len(seq), H, D), np.float32)
        for i in range(len(seq) - 4):
            p = tables[seq[i], pos[i] // page]
            want[i] = q[p, :, pos[i] % page].astype(np.float32) * s[p][:, None]
        assert np.array_equal(got.cpu().numpy(), want.astype(NP[kind]))


def test_append_not_finite_missing_pages_and_unaligned_rows():
    """A page that takes a value that is not finite reads as NaN until it starts afresh; tokens whose page the
    table lacks, and rows before position 0, are passed over; rows at odd offsets."""
    rng = np.random.default_rng(9)
    page, H, D = 16, 2, 32
    new, lens = [20, 5, 40, 6], [30, 3, 40, 6]  # the second has more rows than tokens
    tables, pages = tables_of([max(n, 1) for n in lens], page, rng)
    tables[2, 1] = -1
    tables[2, 2] = pages + 100
    tables = tables[:, :3]
    cache = O.Cache(pages, H, page, D, seed=1)
    T = sum(new)
    rows = rng.standard_normal((T, 2 * H, D + 1)).astype(np.float32)
    rows[3, 0, 5] = np.inf
    rows[8, 2, 7] = np.nan
    pool = pool_of(cache, "heads")
    t = cuda(rows)
    k, v = t[:, :H, 1:], t[:, H:, 1:]
    O.append(cache, rows[:, :H, 1:], rows[:, H:, 1:], starts_of(new), lens, tables)
    Dc.append_noalloc(pool, k, v, cuda(starts_of(new)), cuda(np.array(lens, np.int32)), cuda(tables), stream=stream())
    # positions of a NaN page hold 0; older values stay as they were
    same_cache(pool, cache)
    assert np.isnan(cache.ks).sum() == 1 and np.isnan(cache.vs).sum() == 1
    # one more token keeps it NaN; the page begun afresh is finite again
    one = rng.standard_normal((1, H, D)).astype(np.float32)
    b = int(tables[0, 0])
    Dc.append_noalloc(pool, cuda(one), cuda(one), cuda(np.array([0, 1], np.int32)), cuda(np.array([12], np.int32)),
                      cuda(tables[:1]), stream=stream())
    assert np.isnan(pool.keep[2].cpu().numpy()[b, 0])
    Dc.append_noalloc(pool, cuda(one), cuda(one), cuda(np.array([0, 1], np.int32)), cuda(np.array([1], np.int32)),
                      cuda(tables[:1]), stream=stream())
    assert np.isfinite(pool.keep[2].cpu().numpy()[b]).all()


# ----------------------------------------------------------------- attend ----

class Case:
    def __init__(self, kind, page, hk, group, D, lens, news, layout="heads", seed=0, width=0):
        rng = np.random.default_rng(seed + D + page)
        self.kind, self.lens, self.news = kind, np.array(lens, np.int32), news
        self.tables, pages = tables_of(lens, page, rng, width=width)
        self.cache = O.Cache(pages, hk, page, D, seed=seed)
        self.starts = starts_of(news)
        self.q = (rng.standard_normal((sum(news), hk * group, D)) * 1.5).astype(NP[kind])
        self.layout, self.scale = layout, 1.0 / np.sqrt(D)

    def run(self, causal=True, window=0, work=None, pool=None, q=None, out=None):
        work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda") if work is None else work
        pool = pool or pool_of(self.cache, self.layout)
        q = cuda(self.q) if q is None else q
        out = torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda") if out is None else out
        lse = torch.full(q.shape[:2], 9.0, device="cuda")
        Dc.attend_noalloc(pool, q, cuda(self.starts), cuda(self.lens), cuda(self.tables), out, lse=lse, scale=self.scale,
                          causal=causal, window=window, workspace=work, stream=stream())
        return out.cpu().numpy(), lse.cpu().numpy()

    def check(self, got, causal=True, window=0):
        out, lse = got
        want, wl, mag, vmax = O.attend(self.cache, self.q, self.starts, self.lens, self.tables, self.scale, causal, window)
        empty = np.isneginf(wl)
        assert np.array_equal(np.isneginf(lse), empty) and np.all(out[empty] == 0)
        d = 2.0 ** -20 * mag
        tol = (2 * d + 2.0 ** -18) * vmax
        if self.kind == "f16":
            tol = tol + 2.0 ** -11 * vmax
        tol = tol[..., None] + np.abs(want) * (2.0 ** -11 if self.kind == "f16" else 2.0 ** -22) + 2.0 ** -25
        err = np.abs(out.astype(np.float64) - want)
        assert np.all(err <= tol), "off by %g where %g is allowed" % (err.max(), tol.flat[np.argmax(err - tol)])
        ok = ~empty
        assert np.all(np.abs(lse[ok] - wl[ok]) <= d[ok] + 2.0 ** -20 * (1 + np.abs(wl[ok])))


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("page,hk,group,D,lens,news,layout", [
    (16, 1, 1, 16, [1], [1], "heads"),
    (16, 8, 1, 64, [256], [1], "heads"),
    (64, 2, 4, 128, [1, 0, 17, 64, 65, 700, 128], [1, 1, 1, 1, 1, 1, 0], "heads"),
    (32, 3, 3, 96, [5, 100, 333, 0], [2, 6, 1, 3], "tokens"),
    (128, 1, 16, 80, [130, 50], [1, 2], "tokens"),
    (256, 2, 5, 256, [300, 1000], [1, 3], "heads"),
    (16, 2, 8, 256, [77, 90], [1, 1], "tokens"),
    (16, 1, 7, 192, [500], [9], "heads"),
    (64, 2, 2, 112, [150, 40], [150, 33], "heads"),
    (32, 1, 8, 128, [200, 64, 300], [200, 1, 130], "tokens"),
    (16, 2, 1, 32, [260], [257], "heads")])
def test_attend(kind, page, hk, group, D, lens, news, layout):
    c = Case(kind, page, hk, group, D, lens, news, layout, seed=len(lens))
    for causal, window in ((True, 0), (False, 0), (True, 1), (True, 20), (False, 50), (True, 1 << 30)):
        c.check(c.run(causal, window), causal, window)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("page,hk,group,D,lens,news,layout", [
    (16, 1, 1, 16, [17], [17], "heads"),
    (64, 1, 8, 128, [3000], [20], "heads"),
    (16, 2, 3, 128, [400, 129, 1000, 5], [300, 129, 1, 5], "tokens"),
    (128, 1, 5, 256, [500, 64], [200, 64], "heads"),
    (256, 2, 2, 240, [700], [90], "tokens"),
    (32, 1, 16, 64, [260, 1], [260, 1], "heads"),
    (64, 3, 1, 80, [128, 127, 0, 129], [128, 127, 130, 129], "tokens"),
    (16, 1, 4, 48, [2500, 33], [40, 33], "heads")])
def test_attend_prompts(kind, page, hk, group, D, lens, news, layout):
    """Many rows a sequence: tiles of 128 rows that end inside a token's heads, units cut between blocks, rows of
    sequences that have none to see."""
    c = Case(kind, page, hk, group, D, lens, news, layout, seed=7)
    work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    pool = pool_of(c.cache, layout)
    for causal, window in ((True, 0), (False, 0), (True, 100)):
        got = c.run(causal, window, work=work, pool=pool)
        c.check(got, causal, window)
        again = c.run(causal, window, work=work, pool=pool)
        assert again[0].tobytes() == got[0].tobytes() and again[1].tobytes() == got[1].tobytes()
    assert int(work[:8192].to(torch.int32).sum()) == 0


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("hk,group,D,lens", [(1, 8, 128, [40001]), (2, 4, 64, [30000, 3]), (1, 1, 256, [9000]),
                                             (1, 16, 128, [20000, 11000])])
def test_attend_long_contexts_split_and_joined(kind, hk, group, D, lens):
    """Units cut among many blocks, more than one level of joining; the workspace's counters are left at zero, and
    the same call gives the same bits."""
    c = Case(kind, 16, hk, group, D, lens, [1] * len(lens))
    work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    pool = pool_of(c.cache, "heads")
    first = c.run(work=work, pool=pool)
    c.check(first)
    assert int(work[:8192].to(torch.int32).sum()) == 0
    for _ in range(5):
        again = c.run(work=work, pool=pool)
        assert again[0].tobytes() == first[0].tobytes() and again[1].tobytes() == first[1].tobytes()


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_attend_more_rows_than_tokens_holes_and_short_tables(kind):
    """Rows before position 0 see nothing; pages the table lacks are passed over, all of a row's among them; a table
    shorter than the sequence ends it."""
    c = Case(kind, 16, 2, 2, 64, [3, 100, 64, 200], [7, 2, 1, 1])
    c.tables[1, 2] = -1
    c.tables[1, 4] = 1 << 20
    c.tables[2, :] = -1
    c.tables = np.ascontiguousarray(c.tables[:, :9])  # the last holds 144 of its 200 tokens
    for causal, window in ((True, 0), (False, 0), (True, 3), (True, 40)):
        c.check(c.run(causal, window), causal, window)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("news", [[1, 1], [40, 1], [150, 200]])
def test_attend_what_a_row_does_not_see_does_not_reach_it(kind, news):
    """Scales that are not numbers in pages beyond a row's position, window or length; rows that see one are NaN."""
    c = Case(kind, 16, 1, 2, 64, [250, 260], news)
    clean = c.run()
    bad = c.tables[0, 250 // 16]  # the first sequence's last page: positions 240..249
    c.cache.ks[bad] = np.nan
    c.cache.vs[bad] = np.nan
    out, lse = c.run()
    n = news[0]
    sees = np.zeros(sum(news), bool)
    sees[:n] = np.arange(250 - n, 250) >= 240
    assert np.isnan(out[sees]).all() and np.isnan(lse[sees]).all()
    assert out[~sees].tobytes() == clean[0][~sees].tobytes() and lse[~sees].tobytes() == clean[1][~sees].tobytes()
    # a page behind the window, and one that no table names
    c.cache.ks[bad] = 0.01
    c.cache.vs[bad] = 0.01
    c.cache.ks[c.tables[1, 0]] = np.nan
    c.cache.vs[c.tables[1, 0]] = np.inf
    spare = sorted(set(range(c.cache.k.shape[0])) - set(c.tables.ravel().tolist()))[0]
    c.cache.vs[spare] = np.nan
    out, lse = c.run(window=30)
    rows = np.arange(c.starts[1], c.starts[2])
    far = rows[(260 - len(rows) + np.arange(len(rows))) - 30 + 1 >= 16]
    assert np.isfinite(out[far]).all() and np.isfinite(lse[far]).all()
    assert np.isfinite(out[:c.starts[1]]).all()


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_attend_extreme_scales_and_scores(kind):
    """Value scales from 1e-30 to 1e4 over a sequence's pages, score gaps past exp's range, zero scales, scores whose
    magnitude rounds: against the 64-bit form by the stated bounds; infinite queries make their own rows NaN."""
    c = Case(kind, 16, 2, 4, 128, [300, 64], [1, 1], seed=5)
    c.cache.vs[:] = (10.0 ** np.linspace(-30, 4, c.cache.vs.size)).reshape(c.cache.vs.shape).astype(np.float32)
    c.cache.vs[c.tables[1, 0]] = 0
    if kind == "f16":
        c.cache.vs = np.minimum(c.cache.vs, np.float32(400))  # results within float16
    c.check(c.run())
    c.cache.vs[:] = 0.02
    c.cache.ks[:] = 30.0
    c.check(c.run())
    c.cache.ks[:] = 0
    c.check(c.run())
    c.cache.ks[:] = 0.02
    clean = c.run()
    c.q[0, 3, 7] = np.inf
    out, lse = c.run()
    assert np.isnan(out[0, 3]).all()
    keep = np.ones(out.shape[:2], bool)
    keep[0, 3] = False
    assert out[keep].tobytes() == clean[0][keep].tobytes()


def test_attend_float32_queries_of_every_magnitude():
    """Rows scaled by powers of ten: float32 queries keep 22 bits whatever their size."""
    c = Case("f32", 32, 2, 4, 64, [150, 70], [3, 1], seed=8)
    c.q *= (10.0 ** np.random.default_rng(0).integers(-30, 3, c.q.shape[:2]))[..., None].astype(np.float32)
    c.q[1, 2] = 0
    c.check(c.run())


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("news", [[1, 1, 1], [90, 1, 140]])
def test_attend_strided_queries_and_results(kind, news):
    """Queries and results as slices of wider rows, heads before tokens; nothing else is written."""
    c = Case(kind, 32, 2, 3, 48, [99, 200, 140], news)
    T, H, D = c.q.shape
    wide = torch.full((T, H + 3, D + 5), 3.0, dtype=torch.from_numpy(c.q).dtype, device="cuda")
    q = wide[:, 1:1 + H, 3:3 + D]
    q.copy_(cuda(c.q))
    hold = torch.full((H, T + 1, D + 2), 5.0, dtype=q.dtype, device="cuda")
    out = hold[:, :T, 1:1 + D].transpose(0, 1)
    got = c.run(q=q, out=out)
    c.check(got)
    hold[:, :T, 1:1 + D] = 5.0
    assert bool((hold == 5.0).all())


def test_attend_rows_outside_the_batch_are_left():
    """Rows past the last sequence's stay as they were; an empty batch and empty activations are no work."""
    c = Case("f16", 16, 1, 2, 32, [20, 30], [1, 2])
    q = cuda(np.concatenate([c.q, c.q[:2]]))
    out = torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda")
    c.run(q=q, out=out)
    assert bool((out[3:] == 9.0).all()) and not bool((out[:3] == 9.0).all())
    work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    Dc.attend_noalloc(pool_of(c.cache, "heads"), q[:0], cuda(np.array([0], np.int32)), cuda(np.zeros(0, np.int32)),
                      cuda(np.zeros((0, 1), np.int32)), out[:0], scale=1.0, workspace=work, stream=stream())


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("lens,news", [([40], [2]), ([40], [70]), ([300, 20], [2, 1])])
def test_attend_buffers_longer_than_the_batch(kind, lens, news):
    """Activations of a fixed, longer buffer: the batch's rows are right, whichever kernel the buffer's length
    suggests, and the others stay."""
    c = Case(kind, 16, 1, 4, 64, [max(a, b) for a, b in zip(lens, news)], news)
    q = cuda(np.concatenate([c.q, np.repeat(c.q[:1], 200, 0)]))
    out = torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda")
    got = c.run(q=q, out=out)
    T = len(c.q)
    c.check((got[0][:T], got[1][:T]))
    assert np.all(got[0][T:] == 9.0) and np.all(got[1][T:] == 9.0)


def test_cache_past_32_bit_offsets():
    """Pages past 2^32 bytes of the cache, written, read back and attended to."""
    page, H, D = 256, 2, 256
    each = H * page * D
    pages = (1 << 32) // each + 40
    k, v = (torch.zeros(pages, H, page, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, H, device="cuda") for _ in range(2))
    pool = Dc.Pool(k, v, ks, vs)
    c = Case("f16", page, H, 4, D, [600], [1])
    ids = np.array([[pages - 1, pages - 20, pages - 3]], np.int32)
    rng = np.random.default_rng(0)
    kv = rng.standard_normal((600, 2 * H, D)).astype(np.float16)
    t = cuda(kv)
    st, ln, tb = cuda(np.array([0, 600], np.int32)), cuda(np.array([600], np.int32)), cuda(ids)
    Dc.append_noalloc(pool, t[:, :H], t[:, H:], st, ln, tb, stream=stream())
    small = O.Cache(3, H, page, D)
    O.append(small, kv[:, :H], kv[:, H:], [0, 600], [600], np.array([[0, 1, 2]]))
    assert np.array_equal(k[ids[0].tolist()].cpu().numpy()[:, :, :88], small.k[:, :, :88])
    assert int(k[: pages - 20].count_nonzero()) == 0
    c.cache, c.tables = small, np.array([[0, 1, 2]], np.int32)
    big, c.tables = c.tables, ids
    got = c.run(pool=pool)
    c.tables = big
    c.check(got)


def test_another_stream_than_the_default():
    """The operators queue on the caller's stream, in its order."""
    s = torch.cuda.Stream()
    rng = np.random.default_rng(2)
    c = Case("f16", 16, 2, 4, 64, [100], [1])
    new = rng.standard_normal((1, 4, 64)).astype(np.float16)
    pool, t = pool_of(c.cache, "heads"), cuda(new)
    work = torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    args = [cuda(c.starts), cuda(c.lens), cuda(c.tables)]
    q, pos = cuda(c.q), cuda(np.array([99], np.int32))
    phases, _ = Dc.rope_phases(64)
    ph = cuda(phases)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        turned, out = torch.empty_like(q), torch.empty_like(q)
        Dc.rope_noalloc(q, pos, ph, turned, stream=s.cuda_stream)
        Dc.append_noalloc(pool, t[:, :2], t[:, 2:], *args, stream=s.cuda_stream)
        Dc.attend_noalloc(pool, turned, *args, out, scale=c.scale, workspace=work, stream=s.cuda_stream)
    s.synchronize()
    O.append(c.cache, new[:, :2], new[:, 2:], c.starts, c.lens, c.tables)
    same_cache(pool, c.cache)
    c.q = turned.cpu().numpy()
    lse = c.run(pool=pool)[1]
    c.check((out.cpu().numpy(), lse))


class Shifted:
    """A tensor's description with an address a byte further on, as a C caller could pass it."""

    def __init__(self, t):
        self.t = t

    def data_ptr(self):
        return self.t.data_ptr() + 1

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_refusals():
    """Arguments that no kernel takes come back as errors, and nothing is written."""
    c = Case("f16", 16, 2, 2, 64, [20], [1])
    q, st, ln, tb = cuda(c.q), cuda(c.starts), cuda(c.lens), cuda(c.tables)
    out, work = torch.zeros_like(q), torch.zeros(Dc.attend_workspace(), dtype=torch.uint8, device="cuda")
    pool = pool_of(c.cache, "heads")

    def refuses(text, f, *a, **k):
        with pytest.raises(ShloError, match=text):
            f(*a, **k)
    at = lambda **k: dict(dict(scale=1.0, workspace=work), **k)  # noqa: E731
    refuses("workspace", Dc.attend_noalloc, pool, q, st, ln, tb, out, **at(workspace=work[:-16]))
    refuses("host memory", Dc.attend_noalloc, pool, q, st.cpu(), ln, tb, out, **at())
    refuses("host memory", Dc.attend_noalloc, pool, q, st, ln, tb, out, **at(workspace=work.cpu()))
    refuses("host memory", Dc.rope_noalloc, q.cpu(), ln, ln.long(), out)
    refuses("misaligned", Dc.attend_noalloc, pool, q, st, Shifted(ln), tb, out, **at())
    refuses("not carried", Dc.attend_noalloc, pool, q.bfloat16(), st, ln, tb, out, **at())
    refuses("window", Dc.attend_noalloc, pool, q, st, ln, tb, out, **at(window=-1))
    refuses("shape and type", Dc.attend_noalloc, pool, q, st, ln, tb, out.float(), **at())
    refuses("multiple", Dc.attend_noalloc, pool, q[:, :3], st, ln, tb, out[:, :3], **at())
    refuses("width", Dc.attend_noalloc, pool, q[..., :32], st, ln, tb, out[..., :32], **at())
    refuses("starts", Dc.attend_noalloc, pool, q, st[:1], ln, tb, out, **at())
    refuses("int32", Dc.attend_noalloc, pool, q, st.long(), ln, tb, out, **at())
    refuses("strided", Dc.attend_noalloc, pool, q.transpose(1, 2).contiguous().transpose(1, 2), st, ln, tb, out, **at())
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8, device="cuda")
    s = torch.zeros(4, 2, device="cuda")
    for bad, text in (((k[:, :, :15], k[:, :, :15], s, s), "tokens a page"), ((k[..., :40], k[..., :40], s, s), "head width"),
                      ((k[..., 1:33], k[..., 1:33], s, s), "16 bytes")):
        p = Dc.Pool(*bad)
        qq = torch.zeros(1, 2, bad[0].shape[3], dtype=torch.float16, device="cuda")
        refuses(text, Dc.attend_noalloc, p, qq, st, ln, tb, qq, **at())
        refuses(text, Dc.append_noalloc, p, qq, qq, st, ln, tb)
    refuses("cache", Dc.Pool, k, k[:3], s, s)
    refuses("cache", Dc.Pool, k.float(), k, s, s)
    refuses("cache", Dc.Pool, k, k, s[:, :1], s)
    refuses("kv_append", Dc.append_noalloc, pool, q, q, st, ln, tb)
    refuses("kv_gather", Dc.gather_noalloc, pool, tb, st, st[:1], out, out)
    refuses("out is not", Dc.rope_noalloc, q, ln, torch.zeros(8, dtype=torch.int64, device="cuda"), out[:, :2])
    refuses("turned", Dc.rope_noalloc, q, ln, torch.zeros(33, dtype=torch.int64, device="cuda"), out)
    refuses("positions", Dc.rope_noalloc, q, torch.zeros(2, dtype=torch.int32, device="cuda"),
            torch.zeros(8, dtype=torch.int64, device="cuda"), out)
    assert not bool(out.any())
