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


def fwd(L, dtype=3, n=64, B=2, H=4, Hk=2, dh=64, W=16, S=0, lse=None):
    return L.lib.circatt_sliding_fwd(dtype, n, B, H, Hk, dh, W, S, 0.125, P, H * dh, 0, P, Hk * dh, 0, P, Hk * dh, 0, None, FAR,
                                     None, lse, None)


def bwd(L, dtype=3, n=64, B=2, H=4, Hk=2, dh=64, W=16, S=0):
    return L.lib.circatt_sliding_bwd(dtype, n, B, H, Hk, dh, W, S, 0.125, P, H * dh, 0, P, Hk * dh, 0, P, Hk * dh, 0, None, P,
                                     None, P, P, H * dh, 0, FAR, FAR, FAR, P, 1 << 60, None)


def test_launches_of_too_many_threads_are_refused(L):
    """2^24 workgroups of 256 threads, or 2^23 of 512, and a workgroup at least for
    each signal and head of keys."""
    many = dict(n=1, H=1, Hk=1, dh=8)
    expect(L, fwd(L, B=1 << 24, **many), -2, "threads")
    expect(L, fwd(L, B=(1 << 24) - 7, **many), -2, "threads")  # a multiple of 8 is launched
    # what the forward could do and the backward could not: refused before training
    expect(L, fwd(L, B=1 << 23, lse=P, **many), -2, "threads")
    expect(L, bwd(L, B=1 << 23, **many), -2, "threads")
    size = L.lib.circatt_sliding_bwd_workspace_bytes
    assert size(3, 1, 1 << 23, 1, 1, 8, 16, 0) == -1
    assert size(3, 1, (1 << 23) - 8, 1, 1, 8, 16, 0) > 0
    assert size(3, 300, 50000, 4, 2, 64, 3, 40) > 0
    # long ones: the keys' partial sums would not be the largest launch
    assert size(3, 1 << 20, 64, 1, 1, 8, 16, 100) > 0


def test_paged_append_and_rotary_launches_are_refused(L):
    rc = L.lib.circatt_paged_attention(3, 1 << 30, 1, 1, 1, 8, 16, 0, 0.125, P, 8, P, P, 10, 16, 128, 8, P, 8, 8, P, P, FAR, 1,
                                       P, 1 << 60, None)
    expect(L, rc, -1, "sizes")
    rc = L.lib.circatt_paged_attention(3, (1 << 30) - 1, 65535, 1, 1, 8, 16, 0, 0.125, P, 8, P, P, 10, 16, 128, 8, P, 8, 8, P, P,
                                       FAR, 1, P, 1 << 60, None)
    expect(L, rc, -2, "threads")
    rc = L.lib.circatt_paged_append(3, 1 << 26, 1, 8, P, 8, P, 8, P, P, 10, 16, 128, 8, P, 8, 8, P, P, None)
    expect(L, rc, -2, "threads")
    expect(L, rotary(L, n=(1, 1, 1), tokens=1, nb=1 << 24, H=1, dh=64, x_row=64), -2, "threads")
    expect(L, rotary(L, n=(1, 1, 1), tokens=1, nb=1 << 24, H=1, dh=66, x_row=66), -2, "threads")


def test_windows_and_sinks_beyond_64_bits_hold_every_token():
    from circulant_attention import tokens
    for W in (1 << 31, (1 << 63) + 5, (1 << 64) + 5, 10 ** 30):
        assert tokens._window(W, W, None, 64) == (1 << 30, 1 << 30, 0.125)
    assert tokens._window((1 << 30) - 1, 3, 0.5, 64) == ((1 << 30) - 1, 3, 0.5)
    for W, S in ((-(1 << 64) + 5, 0), (5, -(1 << 64) + 5)):
        with pytest.raises(AssertionError):
            tokens._window(W, S, None, 64)


@pytest.mark.parametrize("heads", [(0, None), (-4, None), (4, 0), (4, -2)])
def test_block_without_heads(heads):
    import circulant_attention as ca
    with pytest.raises(AssertionError, match="divisible"):
        ca.SlidingAttBlock(32, 8, *heads)


def at(address):
    return ctypes.c_void_p(address)


# q is 2 signals of 64 rows of 256 channels (65536 bytes), k and v of 128 (32768), lse 2048 bytes
Q, K, V, Y, REST, LSE, DY, DQ, DK, DV, WORK = (0x100000 * i for i in range(1, 12))


def sliding(L, **where):
    w = dict(q=Q, k=K, v=V, y=Y, rest=REST, lse=LSE)
    w.update(where)
    return L.lib.circatt_sliding_fwd(3, 64, 2, 4, 2, 64, 16, 0, 0.125, at(w["q"]), 256, 64 * 256, at(w["k"]), 128, 64 * 128,
                                     at(w["v"]), 128, 64 * 128, None, at(w["y"]), at(w["rest"]), at(w["lse"]), None)


@pytest.mark.parametrize("where", [dict(y=Q), dict(y=Q + 65536 - 16), dict(y=K - 65536 + 16), dict(y=V + 32768 - 16),
                                   dict(rest=Q + 16), dict(rest=Y + 65536 - 16), dict(lse=Y + 16), dict(lse=V + 32752)])
def test_forward_results_over_arguments(L, where):
    expect(L, sliding(L, **where), -1, "must not overlap")


def sliding_bwd(L, **where):
    w = dict(dq=DQ, dk=DK, dv=DV, work=WORK, dy=DY)
    w.update(where)
    return L.lib.circatt_sliding_bwd(3, 64, 2, 4, 2, 64, 16, 0, 0.125, at(Q), 256, 64 * 256, at(K), 128, 64 * 128, at(V), 128,
                                     64 * 128, None, at(Y), at(REST), at(LSE), at(w["dy"]), 256, 64 * 256, at(w["dq"]),
                                     at(w["dk"]), at(w["dv"]), at(w["work"]), 1 << 40, None)


@pytest.mark.parametrize("where", [dict(dq=DY), dict(dq=Q), dict(dq=Y + 65520), dict(dk=K), dict(dv=V + 16), dict(dv=DK),
                                   dict(dk=DQ + 65520), dict(work=LSE), dict(work=DV + 32752), dict(dq=REST - 65520)])
def test_backward_results_over_arguments(L, where):
    expect(L, sliding_bwd(L, **where), -1, "must not overlap")


@pytest.mark.parametrize("y", [0x10000, 0x10010, 0x10000 + 128 * 512 - 16, 0x10000 - 128 * 512 + 16])
def test_rotary_result_over_its_argument(L, y):
    """2 x 64 tokens of 512 bytes."""
    expect(L, rotary(L, y=at(y)), -1, "alias")
