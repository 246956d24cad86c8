"""The decoder's bookkeeping, without a GPU: what it refuses, and what a step that fails leaves."""
import numpy as np
import pytest

from shlo import decoder as Dd
from shlo._lib import ShloError


@pytest.fixture
def decoder(monkeypatch):
    """A decoder whose arrays are numpy's and whose layers are the test's."""
    monkeypatch.setattr(Dd.M, "of_numpy", lambda a: a)
    monkeypatch.setattr(Dd.M, "to_numpy", lambda a: a)
    monkeypatch.setattr(Dd.M, "reshape", lambda a, shape: a.reshape(shape))
    m = Dd.Decoder.__new__(Dd.Decoder)
    m.cfg, m.free, m.seen = Dd.Config(layers=2, d=8, heads=2, kv_heads=1, page_tokens=4), list(range(10))[::-1], []

    def layer(h, li, t, at, batch):
        m.seen.append((li, t, at.copy(), [b.copy() for b in batch]))
        return h + 1
    m._layer = layer
    return m


def tokens(n, d=8):
    return np.arange(n * d, dtype=np.float32).reshape(n, d)


def test_a_sequence_named_twice_is_refused(decoder):
    a, _ = decoder.start(tokens(3))
    pages, free, n = list(a.pages), list(decoder.free), len(decoder.seen)
    with pytest.raises(ShloError, match="twice"):
        decoder.step([(a, tokens(1)), (Dd.Sequence(), tokens(2)), (a, tokens(3))])
    assert (a.tokens, a.pages, decoder.free, len(decoder.seen)) == (3, pages, free, n)


def test_a_step_that_fails_leaves_lengths_and_pages(decoder):
    a, _ = decoder.start(tokens(3))
    b, layer = Dd.Sequence(), decoder._layer
    before = (a.tokens, list(a.pages), list(decoder.free))

    def broken(h, li, t, at, batch):
        if li == 1:
            raise ShloError("layer")
        return h
    decoder._layer = broken
    with pytest.raises(ShloError, match="layer"):
        decoder.step([(a, tokens(6)), (b, tokens(5))])
    assert (a.tokens, a.pages, decoder.free) == before and (b.tokens, b.pages) == (0, [])
    decoder._layer = layer
    decoder.step([(a, tokens(6)), (b, tokens(5))])
    assert (a.tokens, b.tokens) == (9, 5) and sorted(a.pages + b.pages + decoder.free) == list(range(10))


def test_steps_without_tokens(decoder):
    a, _ = decoder.start(tokens(4))
    before = (a.tokens, list(a.pages), list(decoder.free), len(decoder.seen))
    assert decoder.step([]).shape == (0, 8)
    assert decoder.step([(a, tokens(0)), (Dd.Sequence(), tokens(0))]).shape == (0, 8)
    assert (a.tokens, a.pages, decoder.free, len(decoder.seen)) == before


def test_a_step_lays_its_batch_out(decoder):
    a, y = decoder.start(tokens(5))
    assert np.array_equal(y, tokens(5) + 2)
    b = Dd.Sequence()
    decoder.step([(b, tokens(1)), (a, tokens(4))])
    li, t, at, (starts, lens, tables) = decoder.seen[-1]
    assert (li, t) == (1, 5) and at.tolist() == [0, 5, 6, 7, 8]
    assert starts.tolist() == [0, 1, 5] and lens.tolist() == [1, 9] and tables.tolist() == [b.pages + [-1, -1], a.pages]
    decoder.stop(a)
    assert len(decoder.free) == 9 and (a.tokens, a.pages) == (0, [])
    with pytest.raises(ShloError, match="pages"):
        decoder.start(tokens(40))
    assert len(decoder.free) == 9
