"""The decoder's forks and searches, without a GPU: which pages are shared, copied, freed, and which texts come out."""
import numpy as np
import pytest

import decode8_oracle as O8
from shlo import decoder as Dd
from shlo._lib import ShloError


class FakeCache:
    """Which tokens a page holds, as the device's caches would."""

    def __init__(self, pages):
        self.pages, self.calls = [[] for _ in range(pages)], 0

    def fork(self, tables, lens, parents, fresh):
        self.calls += 1
        seen = set()
        for i, p in enumerate(parents):
            if lens[p] % 4 and p in seen:
                self.pages[fresh[i]] = list(self.pages[tables[p, lens[p] // 4]])
            seen.add(p)
        return tables, lens


@pytest.fixture
def decoder(monkeypatch):
    """Arrays are numpy's; a layer writes its tokens (the rows' first value) into the pages and gives back, of every
    row, the sum over its whole text as the cache holds it: a page that two sequences write into shows."""
    monkeypatch.setattr(Dd.M, "of_numpy", lambda a: a)
    monkeypatch.setattr(Dd.M, "to_numpy", lambda a: a)
    monkeypatch.setattr(Dd.M, "reshape", lambda a, shape: a.reshape(shape))
    m = Dd.Decoder.__new__(Dd.Decoder)
    m.cfg = Dd.Config(layers=1, d=8, heads=2, kv_heads=1, page_tokens=4, vocab=11)
    m.free, m.shared, m.caches = list(range(40))[::-1], {}, [FakeCache(40)]
    m.embed = np.zeros((11, 8), np.float32)
    m.embed[:, 0] = np.arange(11)

    def layer(h, li, t, at, batch):
        starts, lens, tables = batch
        out, pages = np.zeros_like(h), m.caches[0].pages
        for s in range(len(lens)):
            for i in range(starts[s], starts[s + 1]):
                text = pages[tables[s, at[i] // 4]]
                del text[at[i] % 4:]
                text.append(float(h[i, 0]))
                whole = [v for p in tables[s] if p >= 0 for v in pages[p]][:at[i] + 1]
                out[i, 0] = sum((j + 1) * v for j, v in enumerate(whole))
        return out
    m._layer = layer
    m._dense = lambda y, *_: logits(y[:, 0])
    monkeypatch.setattr(Dd.D, "beam_select", lambda z, s, keep, ended, end_token: tuple(
        a.astype(d) for a, d in zip(O8.beam(z, s, keep, ended, end_token), (np.float32, np.int32, np.int32))))
    return m


def logits(key):
    return np.sin(np.outer(key * 1.7 + 1, np.arange(11) + 1)).astype(np.float32) * 2


def expected(prompt, beams, steps, end):
    beam = [(0.0, [], False)]
    for _ in range(steps):
        z = np.concatenate([logits(np.array([sum((j + 1) * v for j, v in enumerate(list(prompt) + t))], np.float32)) for _, t, _ in beam])
        s = np.array([[np.float32(b[0]) for b in beam]], np.float32)
        got = O8.beam(z, s, beams, np.array([[b[2] for b in beam]], np.int32), end)
        beam = [(np.float32(a), beam[p][1] + ([] if beam[p][2] else [int(t)]), beam[p][2] or t == end)
                for a, p, t in zip(*(g[0] for g in got)) if p >= 0]
        if all(b[2] for b in beam):
            break
    return beam


@pytest.mark.parametrize("beams,steps,end,n", [(1, 9, -1, 3), (3, 14, -1, 5), (4, 10, 7, 4), (6, 12, 2, 8), (20, 3, -1, 2)])
def test_search_is_the_plain_one(decoder, beams, steps, end, n):
    prompt = list(range(1, n + 1))
    decoder.free, decoder.caches = list(range(400))[::-1], [FakeCache(400)]
    got, want = decoder.search(prompt, beams, steps, end), expected(prompt, beams, steps, end)
    assert [t for _, t in got] == [t for _, t, _ in want]
    assert np.allclose([a for a, _ in got], [a for a, _, _ in want], rtol=2.0 ** -20)
    assert sorted(decoder.free) == list(range(400)) and not any(decoder.shared.values())


def test_fork_shares_and_copies(decoder):
    s, _ = decoder.start(decoder.embed[[1, 2, 3, 4, 5, 6]])
    full, last = s.pages
    a, b, c = decoder.fork([s], [0, 0, 0])
    assert (s.tokens, s.pages) == (0, []) and all(r.tokens == 6 and r.pages[0] == full for r in (a, b, c))
    assert a.pages[1] == last and len({r.pages[1] for r in (a, b, c)}) == 3 and decoder.shared[full] == 2
    assert decoder.caches[0].pages[b.pages[1]] == [5.0, 6.0]
    d, e = decoder.fork([a, b, c], [2, 2])
    assert decoder.shared[full] == 1 and d.pages == [full, d.pages[1]]
    decoder.stop(d)
    assert full not in decoder.free
    decoder.stop(e)
    assert sorted(decoder.free) == list(range(40)) and decoder.fork([], []) == []


def test_fork_of_full_pages_copies_nothing(decoder):
    s, _ = decoder.start(decoder.embed[[1, 2, 3, 4]])
    before = len(decoder.free)
    a, b = decoder.fork([s], [0, 0])
    assert len(decoder.free) == before and a.pages == b.pages
    decoder.step([(a, decoder.embed[[5]]), (b, decoder.embed[[6]])])
    assert a.pages[0] == b.pages[0] and a.pages[1] != b.pages[1]


def test_fork_without_pages_changes_nothing(decoder):
    s, _ = decoder.start(decoder.embed[[1, 2, 3]])
    decoder.free, pages, calls = decoder.free[:1], list(s.pages), decoder.caches[0].calls
    with pytest.raises(ShloError, match="2 pages needed, 1 free"):
        decoder.fork([s], [0, 0, 0])
    assert (s.tokens, s.pages, len(decoder.free), decoder.caches[0].calls) == (3, pages, 1, calls) and not decoder.shared


def test_search_that_fails_frees_its_pages(decoder):
    layer, seen = decoder._layer, []

    def broken(*a):
        seen.append(1)
        if len(seen) > 3:
            raise ShloError("layer")
        return layer(*a)
    decoder._layer = broken
    with pytest.raises(ShloError, match="layer"):
        decoder.search([1, 2, 3], 3, 9)
    assert sorted(decoder.free) == list(range(40)) and not any(decoder.shared.values())
    for prompt in ([], [11], [3, -1]):
        with pytest.raises(ShloError, match="prompt"):
            decoder.search(prompt, 3, 9)
    decoder.cfg = Dd.Config()
    with pytest.raises(ShloError, match="vocabulary"):
        decoder.search([1], 2, 3)


def test_weights_without_the_new_parts_are_as_before():
    a, b = Dd.init_weights(Dd.Config(), 3), Dd.init_weights(Dd.Config(norm_heads=True, vocab=7), 3)
    assert set(b) - set(a) == {"l0_gq", "l0_gk", "l1_gq", "l1_gk", "embed", "head", "chead"}
    assert all(np.array_equal(a[k], b[k]) for k in a)
