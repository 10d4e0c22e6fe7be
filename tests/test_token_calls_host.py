"""Refusals of the token operators' calls, on the CPU; no kernel runs."""
import ctypes
import math

import pytest
import torch

P = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first
FAR = ctypes.c_void_p(0x7000000000)


@pytest.fixture(scope="module")
def L():
    from circulant_attention import _lib
    return _lib


def expect(L, rc, code, fragment):
    assert rc == code, (rc, L.lib.circatt_last_error())
    assert fragment in L.lib.circatt_last_error().decode(), L.lib.circatt_last_error()


def rotary(L, base=1e4, rest=0.0, n=(8, 8, 1), tokens=64, nb=2, H=4, dh=64, p=(16, 16, 0), x=P, x_row=256, positions=None,
           pos_batch=0, y=FAR):
    return L.lib.circatt_axial_rotary_wide(3, 0, 0, 2, *n, tokens, nb, H, dh, *p, base, rest, x, x_row, positions,
                                           pos_batch, y, None)


@pytest.mark.parametrize("args", [dict(base=0.0), dict(base=-1.0), dict(base=math.inf), dict(base=math.nan),
                                  dict(rest=math.nan), dict(rest=math.inf), dict(base=1.0, rest=-1.0)])
def test_rotary_bases(L, args):
    expect(L, rotary(L, **args), -1, "base")
