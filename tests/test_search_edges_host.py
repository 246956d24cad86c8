"""The decoder's forks and searches at their edges, without a GPU."""
import numpy as np
import pytest

from shlo._lib import ShloError
from test_search_host import decoder, expected  # noqa: F401


def test_forks_that_name_no_row_or_one_twice(decoder):  # noqa: F811
    """Refused before anything changes: a parent behind the rows or before them (the last of a list, in Python), and a
    row under two numbers, whose last page two sequences would write into."""
    a, _ = decoder.start(decoder.embed[[1, 2, 3, 4, 5, 6]])
    b, _ = decoder.start(decoder.embed[[7, 8]])
    before = list(decoder.free), list(a.pages), list(b.pages), decoder.caches[0].calls
    for rows, parents in (([a, b], [0, -1]), ([a, b], [2]), ([a, b], [-2, 0]), ([], [0]), ([a, a], [0, 1]), ([a, b, a], [1])):
        with pytest.raises(ShloError):
            decoder.fork(rows, parents)
        assert (list(decoder.free), a.pages, b.pages, decoder.caches[0].calls) == before and not decoder.shared
    c, d = decoder.fork([a, b], np.array([1, 1]))
    assert c.tokens == d.tokens == 2 and a.tokens == 0


@pytest.mark.parametrize("prompt,beams,steps,end,pages", [([1, 2, 3, 4], 5, 1, -1, 1), ([1, 2], 3, 1, -1, 1), ([1, 2, 3, 4], 3, 5, -1, 6),
                                                          ([5], 1, 4, -1, 1), ([1, 2, 3], 2, 2, -1, 2)])
def test_the_last_step_takes_no_pages(decoder, prompt, beams, steps, end, pages):  # noqa: F811
    """The last tokens are chosen, not computed on: a search runs in the pages that its steps before need. (Pages of four
    tokens: a prompt of 4 has one, three beams one each for the four tokens that are computed on, and a fork copies two while
    the old rows hold theirs; a fifth token would want three more.)"""
    decoder.free = decoder.free[-pages:]
    free = sorted(decoder.free)
    got, want = decoder.search(prompt, beams, steps, end), expected(prompt, beams, steps, end)
    assert [t for _, t in got] == [t for _, t, _ in want]
    assert sorted(decoder.free) == free and not any(decoder.shared.values())
