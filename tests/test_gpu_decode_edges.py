"""The decoder operators on the GPU where a batch or its addresses are unusual; the tolerances of
tests/test_gpu_decode.py, whose cases these use."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from shlo import decode as Dc  # noqa: E402
from shlo import mlx as M  # noqa: E402
from test_gpu_decode import Case, cuda  # noqa: E402


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
