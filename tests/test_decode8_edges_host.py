"""What the launch functions of the norm with rotation, the products in 8 bits, beam search and the cache's reordering
refuse, and what their Python forms do, where no GPU is needed: the checks come before anything is launched or read."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from shlo import mlx as M  # noqa: E402
from shlo._lib import MUL_MAT8_ARGS, load  # noqa: E402

# (with a device what is not refused would run, on addresses where nothing lies)
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls without a device")

SMS = 148
FAR = 1 << 45  # between addresses that share no memory; nothing lies there


def launch(name, *args):
    """The launch function's message, or "" where it refuses nothing (then it fails for want of a device)."""
    L = load()
    f = getattr(L, name)
    f.restype = ctypes.c_int
    assert f(*args) != 0
    said = L.shlo_last_error().decode()
    return "" if "CUDA" in said or "driver" in said else said


def mul_mat8(**change):
    a = dict(x=FAR, x_row=64, x_scale=2 * FAR, w=3 * FAR, w_row=64, w_scale=4 * FAR, bias=5 * FAR, y=6 * FAR, y_row=100, work=7 * FAR,
             work_bytes=1 << 30, rows=5, n=64, m=100, dtype=M.dtF32, x_dtype=M.dtF32)
    a.update(change)
    return MUL_MAT8_ARGS.pack(*a.values())


def product(entry, **change):
    args = mul_mat8(x_dtype=M.dtI8 if entry == "mul_mat8" else M.dtF32, **change)
    if entry == "mul_mat8":
        return launch("_ZN4shlo15launch_mul_mat8ERK18shlo_mul_mat8_argsbPiiP11CUstream_st", args, False, None, SMS, None)
    return launch("_ZN4shlo14launch_linear8ERK18shlo_mul_mat8_argsPiiP11CUstream_st", args, None, SMS, None)


@pytest.mark.parametrize("entry", ["mul_mat8", "linear8"])
@pytest.mark.parametrize("rows", [1, 4, 100])
def test_more_channels_than_are_counted(entry, rows):
    """The kernels' 32-bit counts of channels go on for a grid's or a tile's channels behind the last."""
    assert product(entry, rows=rows) == ""
    for m in ((1 << 30) + 1, (1 << 31) - 4736, (1 << 31) - 1):
        assert "at most 2^30" in product(entry, rows=rows, m=m, y_row=m)
