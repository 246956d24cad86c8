"""Checks of arguments that need no GPU: the norm with rotation, the products in 8 bits, beam search."""
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import decode8_oracle as O8  # noqa: E402
from shlo import _lib  # noqa: E402
from shlo import decode as Dc  # noqa: E402
from shlo._lib import ShloError  # noqa: E402
from test_decode_devices import On  # noqa: E402

ENTRIES = ["norm_rope", "norm_rope_grad", "quantise_rows", "mul_mat8", "linear8", "beam_select", "kv_fork"]


@pytest.fixture
def calls(monkeypatch):
    made = []

    def entry(name):
        return lambda *a: made.append(name) or 0
    lib = types.SimpleNamespace(shlo_cuda_device=lambda: 0, **{"shlo_%s_noalloc" % n: entry(n) for n in ENTRIES})
    monkeypatch.setattr(Dc, "load", lambda: lib)
    return made


def operands(other=None, **change):
    f16, i32, i8 = torch.float16, torch.int32, torch.int8
    t = dict(x=torch.zeros(3, 4, 16, dtype=f16), dy=torch.zeros(3, 4, 16, dtype=f16), y=torch.zeros(3, 4, 16, dtype=f16),
             pos=torch.zeros(3, dtype=i32), phases=torch.zeros(8, dtype=torch.int64), wq=torch.ones(16, dtype=f16), wk=torch.ones(16, dtype=f16),
             dq=torch.zeros(16), dk=torch.zeros(16), work=torch.zeros(1 << 20, dtype=torch.uint8),
             a=torch.zeros(5, 32, dtype=f16), q=torch.zeros(5, 32, dtype=i8), s=torch.zeros(5), w=torch.zeros(7, 32, dtype=i8),
             ws=torch.zeros(7), bias=torch.zeros(7), out=torch.zeros(5, 7, dtype=f16),
             z=torch.zeros(6, 50, dtype=f16), scores=torch.zeros(2, 3), next=torch.zeros(2, 4), parents=torch.zeros(2, 4, dtype=i32),
             tokens=torch.zeros(2, 4, dtype=i32), ended=torch.zeros(2, 3, dtype=i32),
             k=torch.zeros(9, 2, 16, 16, dtype=i8), v=torch.zeros(9, 2, 16, 16, dtype=i8), ks=torch.zeros(9, 2), vs=torch.zeros(9, 2),
             tables=torch.zeros(6, 2, dtype=i32), lens=torch.zeros(6, dtype=i32), fresh=torch.zeros(8, dtype=i32),
             tables2=torch.zeros(8, 2, dtype=i32), lens2=torch.zeros(8, dtype=i32), q_heads=3)
    t.update(change)
    return {n: On(x, 1 if n == other else 0) if torch.is_tensor(x) else x for n, x in t.items()}


def run(t):
    w = dict(q_heads=t["q_heads"], q_weight=t["wq"], k_weight=t["wk"], eps=1e-6)
    Dc.norm_rope_noalloc(t["x"], t["pos"], t["phases"], t["y"], **w)
    Dc.norm_rope_grad_noalloc(t["x"], t["dy"], t["pos"], t["phases"], t["y"], t["dq"], t["dk"], workspace=t["work"], **w)
    Dc.quantise_rows_noalloc(t["a"], t["q"], t["s"])
    Dc.mul_mat8_noalloc(t["q"], t["s"], t["w"], t["ws"], t["out"], bias=t["bias"])
    Dc.linear8_noalloc(t["a"], t["w"], t["ws"], t["out"], bias=t["bias"], workspace=t["work"])
    Dc.beam_select_noalloc(t["z"], t["scores"], t["next"], t["parents"], t["tokens"], ended=t["ended"], workspace=t["work"])
    Dc.fork_noalloc(Dc.Pool(t["k"], t["v"], t["ks"], t["vs"]), t["tables"], t["lens"], t["parents"], t["fresh"], t["tables2"], t["lens2"])


def test_all_are_called(calls):
    run(operands())
    run(operands(wq=None, wk=None, bias=None, ended=None, dq=None, dk=None, q_heads=0))
    assert calls == 2 * ENTRIES


FIRST = dict(x=0, y=0, pos=0, phases=0, wq=0, wk=0, dy=1, dq=1, dk=1, work=1, a=2, q=2, s=2, w=3, ws=3, bias=3, out=3, z=5, scores=5,
             next=5, parents=5, tokens=5, ended=5, k=6, v=6, ks=6, vs=6, tables=6, lens=6, fresh=6, tables2=6, lens2=6)


@pytest.mark.parametrize("name", sorted(FIRST))
def test_a_tensor_of_another_device(calls, name):
    with pytest.raises(ShloError, match="device 1"):
        run(operands(name))
    assert calls == ENTRIES[:FIRST[name]]


@pytest.mark.parametrize("name", sorted(FIRST))
def test_a_tensor_in_host_memory(calls, name):
    t = operands()
    t[name] = t[name].t
    with pytest.raises(ShloError, match="host memory"):
        run(t)
    assert calls == ENTRIES[:FIRST[name]]


@pytest.mark.parametrize("at,change", [
    (0, dict(x=torch.zeros(3, 4, 16, dtype=torch.float64))), (0, dict(x=torch.zeros(3, 64))), (0, dict(y=torch.zeros(3, 4, 16))),
    (0, dict(x=torch.zeros(3, 4, 32, dtype=torch.float16)[:, :, ::2])), (0, dict(pos=torch.zeros(4, dtype=torch.int32))),
    (0, dict(pos=torch.zeros(3, dtype=torch.int64))), (0, dict(phases=torch.zeros(8))), (0, dict(wq=torch.ones(15))),
    (0, dict(wk=torch.ones(16))), (0, dict(wq=torch.ones(32)[::2], wk=None)), (0, dict(q_heads=5)), (0, dict(q_heads=-1)),
    (1, dict(dy=torch.zeros(3, 4, 16))), (1, dict(dq=torch.zeros(16, dtype=torch.float16))), (1, dict(dk=torch.zeros(17))),
    (2, dict(a=torch.zeros(5, 32, dtype=torch.int8))), (2, dict(q=torch.zeros(5, 31, dtype=torch.int8))), (2, dict(s=torch.zeros(4))),
    (2, dict(q=torch.zeros(1, 32, dtype=torch.int8).expand(5, 32))),
    (3, dict(w=torch.zeros(7, 31, dtype=torch.int8))), (3, dict(ws=torch.zeros(6))), (3, dict(bias=torch.zeros(7, dtype=torch.float16))),
    (3, dict(out=torch.zeros(5, 8, dtype=torch.float16))), (3, dict(out=torch.zeros(5, 7, dtype=torch.int32))),
    (3, dict(out=torch.zeros(1, 7, dtype=torch.float16).expand(5, 7))), (3, dict(w=torch.zeros(7, 64, dtype=torch.int8)[:, ::2])),
    (5, dict(z=torch.zeros(5, 50, dtype=torch.float16))), (5, dict(scores=torch.zeros(6))), (5, dict(parents=torch.zeros(2, 3, dtype=torch.int32))),
    (5, dict(tokens=torch.zeros(2, 4))), (5, dict(ended=torch.zeros(2, 3))), (5, dict(next=torch.zeros(2, 8)[:, ::2])),
    (6, dict(lens=torch.zeros(5, dtype=torch.int32))), (6, dict(fresh=torch.zeros(7, dtype=torch.int32))),
    (6, dict(tables2=torch.zeros(8, 3, dtype=torch.int32))), (6, dict(tables2=torch.zeros(1, 2, dtype=torch.int32).expand(8, 2))),
    (6, dict(lens2=torch.zeros(8))), (6, dict(k=torch.zeros(9, 2, 16, 16)))])
def test_refusals(calls, at, change):
    with pytest.raises(ShloError):
        run(operands(**change))
    assert calls == ENTRIES[:at]


def test_numbers_that_no_field_holds(calls):
    t = operands()
    for end in (1 << 40, -1 << 31 << 1):
        with pytest.raises(ShloError, match="beam_select"):
            Dc.beam_select_noalloc(t["z"], t["scores"], t["next"], t["parents"], t["tokens"], workspace=t["work"], end_token=end)
    assert calls == []


def test_workspace_sizes():
    assert Dc.linear8_workspace(3, 5) >= 3 * 16 + 3 * 4
    assert Dc.beam_workspace(2, 4, 8, 50000) >= 2 * 4 * 8 * 8
    for args in ((-1, 5), (3, 0), (3, 131072)):
        with pytest.raises(ShloError):
            Dc.linear8_workspace(*args)
    for args in ((1, 0, 1, 9), (1, 65, 1, 9), (1, 1, 65, 9), (1, 1, 1, 0), (2000, 64, 1, 9)):
        with pytest.raises(ShloError):
            Dc.beam_workspace(*args)
    assert _lib.load().shlo_beam_workspace(1, 1, 1, 1, None) != 0


def test_the_oracles_ties():
    """Halves of a step go to the even whole number."""
    q, s = O8.quantise(np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, 62.5]], np.float32))
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, 64, 62]] and s[0] == 1.0


def test_descriptors_are_the_headers(tmp_path):
    """The packed descriptors against the C compiler's layout of include/shlo_cuda.h."""
    import os
    import subprocess
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "shlo_cuda.h"\nint main(void) {\n'
                   '  printf("%zu %zu %zu %zu\\n", offsetof(shlo_norm_rope_args, weight_dtype) + 1, offsetof(shlo_mul_mat8_args, x_dtype) + 1,'
                   ' offsetof(shlo_beam_args, dtype) + 1, offsetof(shlo_kv_fork_args, table_pages) + 4);\n'
                   '  printf("%zu %zu %zu\\n", offsetof(shlo_norm_rope_args, tokens), offsetof(shlo_mul_mat8_args, rows),'
                   ' offsetof(shlo_beam_args, seqs));\n  return 0;\n}\n')
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "sizes")], check=True)
    ends, middles = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines()
    packed = (_lib.NORM_ROPE_ARGS, _lib.MUL_MAT8_ARGS, _lib.BEAM_ARGS, _lib.KV_FORK_ARGS)
    assert [int(v) for v in ends.split()] == [a.size for a in packed]
    assert [int(v) for v in middles.split()] == [_lib.struct.calcsize(f) for f in ("PqqPPPPPqqPqqPPPN", "PqPPqPPPqPN", "PqPPPPPPN")]


def test_null_arguments_are_errors():
    L = _lib.load()
    for name in ("norm_rope", "norm_rope_grad", "mul_mat8", "linear8", "beam_select"):
        assert getattr(L, "shlo_%s_noalloc" % name)(None, None) != 0
        assert "null" in L.shlo_last_error().decode()
    assert L.shlo_kv_fork_noalloc(None, None, None) != 0 and "null" in L.shlo_last_error().decode()
