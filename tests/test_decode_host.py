"""The decoder operators' host side: the phases of the rotary positions, and checks that need no GPU."""
import ctypes
import math

import numpy as np
import pytest

from shlo import _lib
from shlo import decode as Dc
from shlo._lib import ShloError


def radians(phases):
    return phases.astype(np.float64) / 2.0 ** 64 * 2 * math.pi


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (18, 1e6), (2048, 1.5)])
def test_phases_are_the_frequencies(rot, base):
    """Within the 64-bit float's own rounding of the formula (a few times 2^-53) and the phase's (2^-65)."""
    phases, factor = Dc.rope_phases(rot, base)
    want = base ** (-2.0 * np.arange(rot // 2) / rot)
    assert factor == 1.0
    assert np.all(np.abs(radians(phases) - want) <= 2.0 ** -48 * want + 2.0 ** -62)


def test_scaled_phases():
    rot, base, by, trained = 128, 10000.0, 8.0, 2048.0
    i = np.arange(rot // 2)
    f = base ** (-2.0 * i / rot)
    plain = radians(Dc.rope_phases(rot, base)[0])
    assert np.allclose(radians(Dc.rope_phases(rot, base, "linear", by)[0]) * by, plain, rtol=2.0 ** -45)
    raised = radians(Dc.rope_phases(rot, base, "base", by)[0])
    assert np.isclose(raised[0], 1.0, rtol=2.0 ** -45) and np.isclose(raised[-1] * by, plain[-1], rtol=2.0 ** -40)
    phases, factor = Dc.rope_phases(rot, base, "ramp", by, trained, 32.0, 1.0)
    got = radians(phases)
    turns = trained * f / (2 * math.pi)
    assert np.isclose(factor, 0.1 * math.log(by) + 1.0, rtol=2.0 ** -22)
    keep = (f / got - 1.0) / (by - 1.0)  # 0 kept .. 1 divided, before the blend's own nonlinearity
    assert np.allclose(got[turns > 40], f[turns > 40], rtol=2.0 ** -45)
    assert np.allclose(got[turns < 0.8] * by, f[turns < 0.8], rtol=2.0 ** -45)
    assert np.all(np.diff(keep) >= -2.0 ** -40)
    got = radians(Dc.rope_phases(rot, base, "blend", by, trained, 4.0, 1.0)[0])
    w = np.clip((turns - 1.0) / 3.0, 0, 1)
    assert np.allclose(got, f / by * (1 - w) + f * w, rtol=2.0 ** -45)


@pytest.mark.parametrize("args", [(0,), (3,), (4096,), (64, 1.0), (64, float("nan")), (64, 1e4, "linear", 0.5),
                                  (64, 1e4, "ramp", 8.0, 0.0), (64, 1e4, "blend", 8.0, 10.0, 1.0, 1.0), (64, 1e4, "other")])
def test_phases_refuse(args):
    with pytest.raises(ShloError):
        Dc.rope_phases(*args)


def test_descriptors_are_the_headers():
    """The ctypes structures against the C declarations' layout (natural alignment on a 64-bit ABI)."""
    assert ctypes.sizeof(_lib.KvPool) == 4 * 8 + 6 * 8 + 3 * 4 + 4
    assert _lib.KvPool.heads.offset == 80 and _lib.KvPool.page_tokens.offset == 88
    assert ctypes.sizeof(_lib.KvBatch) == 3 * 8 + 8 + 3 * 4 + 4
    assert _lib.KvBatch.tokens.offset == 40


def test_null_descriptors_are_errors():
    L = _lib.load()
    assert L.shlo_kv_attend_workspace(None) != 0
    assert L.shlo_kv_append_noalloc(None, None, None, 0, 0, None, 0, 0, 9, None) != 0
    assert "null" in L.shlo_last_error().decode()
