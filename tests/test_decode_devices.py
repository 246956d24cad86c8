"""Where a call's memory lies, without a GPU: tensors of another device than the current one are refused before any
launch."""
import types

import pytest

torch = pytest.importorskip("torch")

from shlo import decode as Dc  # noqa: E402
from shlo._lib import ShloError  # noqa: E402


class On:
    """A host tensor that says that it lies on a GPU."""
    is_cuda = True

    def __init__(self, t, device=0):
        self.t, self.device_index = t, device

    def get_device(self):
        return self.device_index

    def __getattr__(self, name):
        return getattr(self.t, name)


class Plain:
    """One that does not say which."""
    is_cuda = True

    def __init__(self, t):
        self.shape, self.dtype, self.stride, self.data_ptr = t.shape, t.dtype, t.stride, t.data_ptr
        self.numel, self.element_size, self.is_contiguous = t.numel, t.element_size, t.is_contiguous


@pytest.fixture
def calls(monkeypatch):
    """The library with device 0 as the current one, which counts its calls."""
    made = []

    def entry(name):
        return lambda *a: made.append(name) or 0
    names = ["shlo_rope_noalloc", "shlo_kv_append_noalloc", "shlo_kv_gather_noalloc", "shlo_kv_attend_noalloc"]
    lib = types.SimpleNamespace(shlo_cuda_device=lambda: 0, **{n: entry(n) for n in names})
    monkeypatch.setattr(Dc, "load", lambda: lib)
    return made


def operands(wrap):
    f16, i32 = torch.float16, torch.int32
    t = dict(q=torch.zeros(3, 4, 16, dtype=f16), out=torch.zeros(3, 4, 16, dtype=f16), kv=torch.zeros(3, 2, 16, dtype=f16),
             lse=torch.zeros(3, 4), positions=torch.zeros(3, dtype=i32), phases=torch.zeros(8, dtype=torch.int64),
             starts=torch.tensor([0, 3], dtype=i32), lens=torch.tensor([3], dtype=i32), tables=torch.zeros(1, 1, dtype=i32),
             work=torch.zeros(64, dtype=torch.uint8), k=torch.zeros(1, 2, 16, 16, dtype=torch.int8),
             v=torch.zeros(1, 2, 16, 16, dtype=torch.int8), ks=torch.zeros(1, 2), vs=torch.zeros(1, 2))
    return {n: wrap(x, n) for n, x in t.items()}


def run(t):
    pool = Dc.Pool(t["k"], t["v"], t["ks"], t["vs"])
    Dc.rope_noalloc(t["q"], t["positions"], t["phases"], t["out"])
    Dc.append_noalloc(pool, t["kv"], t["kv"], t["starts"], t["lens"], t["tables"])
    Dc.gather_noalloc(pool, t["tables"], t["positions"], t["positions"], t["kv"], t["kv"])
    Dc.attend_noalloc(pool, t["q"], t["starts"], t["lens"], t["tables"], t["out"], lse=t["lse"], scale=1.0, workspace=t["work"])


def test_one_device(calls):
    run(operands(lambda x, n: On(x)))
    run(operands(lambda x, n: Plain(x)))
    assert len(calls) == 8


@pytest.mark.parametrize("name", ["q", "out", "kv", "lse", "positions", "phases", "starts", "lens", "tables", "work", "k",
                                  "v", "ks", "vs"])
def test_a_tensor_of_another_device(calls, name):
    t = operands(lambda x, n: On(x, 1 if n == name else 0))
    with pytest.raises(ShloError, match="device 1"):
        run(t)
    first = {"q": 0, "out": 0, "positions": 0, "phases": 0, "kv": 1, "starts": 1, "lens": 1, "tables": 1, "work": 3, "lse": 3}
    assert len(calls) == first.get(name, 0)


def test_another_device_than_the_current(calls):
    t = operands(lambda x, n: On(x, 2))
    pool = Dc.Pool(t["k"], t["v"], t["ks"], t["vs"])
    for f, a, k in ((Dc.rope_noalloc, (t["q"], t["positions"], t["phases"], t["out"]), {}),
                    (Dc.append_noalloc, (pool, t["kv"], t["kv"], t["starts"], t["lens"], t["tables"]), {}),
                    (Dc.gather_noalloc, (pool, t["tables"], t["positions"], t["positions"], t["kv"], t["kv"]), {}),
                    (Dc.attend_noalloc, (pool, t["q"], t["starts"], t["lens"], t["tables"], t["out"]),
                     dict(scale=1.0, workspace=t["work"]))):
        with pytest.raises(ShloError, match="device 2"):
            f(*a, **k)
    here = operands(lambda x, n: On(x))
    with pytest.raises(ShloError, match="cache on device 2"):
        Dc.append_noalloc(pool, here["kv"], here["kv"], here["starts"], here["lens"], here["tables"])
    assert not calls


def test_host_memory(calls):
    with pytest.raises(ShloError, match="host memory"):
        run(operands(lambda x, n: x))
    assert not calls
