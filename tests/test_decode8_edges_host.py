"""What the launch functions of the norm with rotation, the products in 8 bits, beam search and the cache's reordering
refuse, and what their Python forms do, where no GPU is needed: the checks come before anything is launched or read."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import test_decode8_host as H  # noqa: E402
import test_decode_devices as Hd  # noqa: E402
from shlo import mlx as M  # noqa: E402
from shlo._lib import MUL_MAT8_ARGS, ShloError, load  # noqa: E402
from test_decode8_host import calls  # noqa: E402, F401

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


# ---- of the Python forms ----

@pytest.mark.parametrize("work", [torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 21, dtype=torch.uint8)[::2],
                                  torch.zeros(64, 64)[:, :32]])
def test_workspaces_that_are_not_contiguous(calls, monkeypatch, work):  # noqa: F811
    """Their values are not the bytes that lie behind their first: a value spread over many takes no more room than one."""
    t = H.operands(work=work)
    w = dict(q_heads=3, q_weight=t["wq"], k_weight=t["wk"], eps=1e-6)
    for f in (lambda: H.Dc.norm_rope_grad_noalloc(t["x"], t["dy"], t["pos"], t["phases"], t["y"], t["dq"], t["dk"], workspace=t["work"], **w),
              lambda: H.Dc.linear8_noalloc(t["a"], t["w"], t["ws"], t["out"], workspace=t["work"]),
              lambda: H.Dc.beam_select_noalloc(t["z"], t["scores"], t["next"], t["parents"], t["tokens"], workspace=t["work"])):
        with pytest.raises(ShloError, match="contiguous"):
            f()
    assert calls == []


def test_attention_over_a_workspace_that_is_not_contiguous(monkeypatch):
    made = []
    lib = type("Lib", (), {"shlo_cuda_device": staticmethod(lambda: 0),
                           "shlo_kv_attend_noalloc": staticmethod(lambda *a: made.append(a) or 0)})
    monkeypatch.setattr(H.Dc, "load", lambda: lib)
    t = Hd.operands(lambda x, n: Hd.On(x))
    pool = H.Dc.Pool(t["k"], t["v"], t["ks"], t["vs"])

    def attend(work):
        H.Dc.attend_noalloc(pool, t["q"], t["starts"], t["lens"], t["tables"], t["out"], scale=1.0, workspace=work)
    attend(t["work"])
    assert made[0][-3:] == (t["work"].data_ptr(), 64, 0)
    with pytest.raises(ShloError, match="contiguous"):
        attend(Hd.On(torch.zeros(1, dtype=torch.uint8).expand(1 << 20)))
    assert len(made) == 1
