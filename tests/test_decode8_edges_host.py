"""What the launch functions of the norm with rotation, the products in 8 bits, beam search and the cache's reordering
refuse, and what their Python forms do, where no GPU is needed: the checks come before anything is launched or read."""
import ctypes
import types

import pytest

torch = pytest.importorskip("torch")

import test_decode8_host as H  # noqa: E402
import test_decode_devices as Hd  # noqa: E402
from shlo import mlx as M  # noqa: E402
from shlo._lib import BEAM_ARGS, MUL_MAT8_ARGS, NORM_ROPE_ARGS, ShloError, load  # noqa: E402
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


# Operands of 5 rows of 64 float32 values (or 8-bit ones), 100 channels.
@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("name,at,length", [("x", FAR, 64 * 4), ("w", 3 * FAR, 99 * 64 + 64), ("w_scale", 4 * FAR, 400), ("bias", 5 * FAR, 400),
                                            ("y", 6 * FAR, 400)])
def test_linear8_workspace_in_other_memory(rows, name, at, length):
    need = rows * (64 + 4) + 16
    length += (rows - 1) * {"x": 256, "y": 400}.get(name, 0)
    inside = [at - need // 16 * 16, at, at + (length - 1) // 16 * 16]
    for work in inside:
        assert "workspace shares memory" in product("linear8", rows=rows, work=work, work_bytes=need)
    for work in (at - (need + 15) // 16 * 16, at + (length + 15) // 16 * 16):
        assert product("linear8", rows=rows, work=work, work_bytes=need) == ""
    # (what lies behind the bytes that are needed is the caller's)
    assert product("linear8", rows=rows, work=at - (need + 15) // 16 * 16, work_bytes=1 << 30) == ""


def beam(**change):
    a = dict(logits=FAR, row=1000, scores=2 * FAR, ended=3 * FAR, next=4 * FAR, parents=5 * FAR, tokens=6 * FAR, work=7 * FAR,
             work_bytes=1 << 30, seqs=2, beams=3, keep=4, vocab=1000, end=-1, dtype=M.dtF32)
    a.update(change)
    return launch("_ZN4shlo18launch_beam_selectERK14shlo_beam_argsiP11CUstream_st", BEAM_ARGS.pack(*a.values()), SMS, None)


@pytest.mark.parametrize("at,length", [(FAR, 6 * 4000), (2 * FAR, 24), (3 * FAR, 24), (4 * FAR, 32), (5 * FAR, 32), (6 * FAR, 32)])
def test_beam_workspace_in_other_memory(at, length):
    n = ctypes.c_size_t()
    assert load().shlo_beam_workspace(2, 3, 4, 1000, ctypes.byref(n)) == 0
    need = n.value
    for work in (at, at - need // 8 * 8 + 8, at + length - 8):
        assert "workspace shares memory" in beam(work=work, work_bytes=need)
    for work in (at - (need + 7) // 8 * 8, at + length):
        assert beam(work=work, work_bytes=need) == ""
    assert beam(work=FAR + 4000, work_bytes=need, row=1000 + (need + 3) // 4 * 2) == ""  # between rows


def norm_rope(back, **change):
    a = dict(x=FAR, x_token=4 * 16, x_head=16, positions=2 * FAR, phases=3 * FAR, wq=4 * FAR, wk=5 * FAR, y=6 * FAR, y_token=4 * 16, y_head=16,
             dy=7 * FAR, dy_token=4 * 16, dy_head=16, dq=8 * FAR, dk=9 * FAR, work=10 * FAR, work_bytes=1 << 30, tokens=3, heads=4, dim=16,
             rot=8, q_heads=2, eps=1e-6, factor=1.0, flags=0, dtype=M.dtF32, wtype=M.dtF16)
    a.update(change)
    return launch("_ZN4shlo16launch_norm_ropeERK19shlo_norm_rope_argsbiP11CUstream_st", NORM_ROPE_ARGS.pack(*a.values()), back, SMS, None)


ROWS = 3 * 4 * 16 * 4


@pytest.mark.parametrize("at,length", [(FAR, ROWS), (2 * FAR, 12), (3 * FAR, 32), (4 * FAR, 32), (5 * FAR, 32), (6 * FAR, ROWS), (7 * FAR, ROWS)])
def test_norm_rope_grad_sums_in_other_memory(at, length):
    """The weights' gradients and the workspace in x, positions, phases, the weights, dx, dy, or each other."""
    need = 3 * SMS * 2 * 512 * 8  # (shlo_norm_rope_workspace's)
    assert norm_rope(True, work_bytes=need - 1) != "" and norm_rope(True, work_bytes=need) == ""
    last = at + (length - 1) // 8 * 8
    for name, size in (("dq", 64), ("dk", 64), ("work", need)):
        for p in (at, last, at - size + 8):
            assert "shares memory" in norm_rope(True, **{name: p})
        for p in (at + (length + 7) // 8 * 8, at - size):
            assert norm_rope(True, **{name: p}) == ""
        assert norm_rope(False, **{name: at}) == ""  # (the forward pass has none)
    for name in ("dq", "dk"):
        assert "shares memory" in norm_rope(True, work=9 * FAR if name == "dk" else 8 * FAR)
        assert norm_rope(True, **{name: FAR + 32}, x_head=24, x_token=96) != ""  # in the first head's second half
        assert norm_rope(True, **{name: FAR + 64}, x_head=32, x_token=128) == ""  # between two heads
        assert norm_rope(True, **{name: FAR + 64 - 4 * 32}, x_head=-32, x_token=128) == ""
        assert norm_rope(True, **{name: FAR - 4 * 32}, x_head=-32, x_token=128) != ""


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("name,length", [("positions", 12), ("phases", 32), ("wq", 32), ("wk", 32)])
def test_norm_rope_rows_in_what_is_read(back, name, length):
    for off in (0, 8, ROWS - 8, 8 - length):
        assert "shares memory" in norm_rope(back, **{name: 6 * FAR + off})
    for off in (ROWS, -length - length % 8):
        assert norm_rope(back, **{name: 6 * FAR + off}) == ""
    assert norm_rope(back, **{name: 6 * FAR + 64}, y_head=32, y_token=128) == ""
    assert (norm_rope(back, **{name: 6 * FAR}, rot=0) == "") == (name in ("positions", "phases"))  # (then they are not read)


@pytest.mark.parametrize("back", [False, True])
def test_more_heads_than_are_counted(back):
    for heads in ((1 << 30) + 1, (1 << 31) - 1):
        assert "2^30" in norm_rope(back, tokens=1, heads=heads, dim=1, rot=0, x_head=1, y_head=1, dy_head=1)
    assert norm_rope(back, tokens=1, heads=1 << 30, dim=1, rot=0, x_head=1, y_head=1, dy_head=1) == ""


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


class Wide(H.On):
    """A tensor that says it has other sizes than it has."""

    def __init__(self, t, shape, stride=None):
        super().__init__(t)
        self.shape, self.strides = shape, stride

    def stride(self):
        return self.strides or self.t.stride()


def test_numbers_that_would_be_cut_to_32_bits(calls, monkeypatch):  # noqa: F811
    t = H.operands()
    n = (1 << 32) + 32
    with pytest.raises(ShloError, match="quantise_rows.*32-bit"):
        H.Dc.quantise_rows_noalloc(Wide(t["a"].t, (5, n), (n, 1)), Wide(t["q"].t, (5, n), (n, 1)), t["s"])
    wide = torch.zeros(1, 2, dtype=torch.int32).expand(1 << 31, 2)
    with pytest.raises(ShloError, match="kv_fork"):
        H.Dc.fork_noalloc(H.Dc.Pool(t["k"], t["v"], t["ks"], t["vs"]), H.On(wide), Wide(t["lens"].t, (1 << 31,), (1,)), t["parents"], t["fresh"],
                          t["tables2"], t["lens2"])
    assert calls == []
    monkeypatch.undo()  # (the library itself)
    for args in ((n, 1, 1, 9), (1, n, 1, 9), (1, 1, n, 9), (1, 1, 1, n)):
        with pytest.raises(ShloError):
            H.Dc.beam_workspace(*args)
    with pytest.raises(ShloError):
        H.Dc.linear8_workspace(1, n)
    arr = types.SimpleNamespace(h=None)
    for f in (lambda: H.Dc.beam_select(arr, arr, n), lambda: H.Dc.beam_select(arr, arr, 4, end_token=-n),
              lambda: H.Dc.norm_rope_grad(arr, arr, arr, arr, arr, arr, q_heads=n, eps=1e-6)):
        with pytest.raises(ShloError, match="32-bit"):
            f()
    monkeypatch.setattr(H.Dc.M, "shape", lambda a: (3, 4, 16))
    for q_heads in (-1, 5, n):
        with pytest.raises(ShloError, match="query heads"):
            H.Dc.norm_rope(arr, arr, arr, arr, arr, q_heads=q_heads, eps=1e-6)


@pytest.mark.parametrize("shape", [(), (2, 4, 5), (8, 1, 2), (0,)])
def test_fork_of_more_parents_than_rows(calls, shape):  # noqa: F811
    """The rows' parents are all that there are: not the first of more."""
    t = H.operands()
    args = (H.Dc.Pool(t["k"], t["v"], t["ks"], t["vs"]), t["tables"], t["lens"])
    for parents in (t["parents"], H.On(torch.zeros(8, dtype=torch.int32)), H.On(torch.zeros(2, 4, 1, dtype=torch.int32))):
        H.Dc.fork_noalloc(*args, parents, t["fresh"], t["tables2"], t["lens2"])
    with pytest.raises(ShloError, match="parents"):
        H.Dc.fork_noalloc(*args, H.On(torch.zeros(shape, dtype=torch.int32)), t["fresh"], t["tables2"], t["lens2"])
    assert calls == 3 * ["kv_fork"]
