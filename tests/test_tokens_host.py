"""What the token operators refuse, on the CPU: the C ABI's argument checks,
which precede every launch, and the Python layer's.  No kernel runs."""
import ctypes
import math

import pytest
import torch

import token_model as M

P = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x10008)


@pytest.fixture(scope="module")
def L():
    from circulant_attention import _lib
    return _lib


def expect(L, rc, code, fragment):
    assert rc == code, (rc, L.lib.circatt_last_error())
    assert fragment in L.lib.circatt_last_error().decode(), L.lib.circatt_last_error()


def fwd(L, dtype=3, n=64, B=2, H=4, Hk=2, dh=64, W=16, S=0, scale=0.125, q=P, q_row=256, q_batch=0, k=P, k_row=128,
        k_batch=0, v=P, v_row=128, v_batch=0, lengths=None, y=P, rest=None, lse=None):
    return L.lib.circatt_sliding_fwd(dtype, n, B, H, Hk, dh, W, S, scale, q, q_row, q_batch, k, k_row, k_batch, v, v_row,
                                     v_batch, lengths, y, rest, lse, None)


@pytest.mark.parametrize("args,code,fragment", [
    (dict(dtype=1), -2, "dtype"), (dict(dtype=9), -2, "dtype"),
    (dict(H=4, Hk=3), -1, "divisible by kv_heads"), (dict(H=0), -1, "head counts"), (dict(Hk=0), -1, "head counts"),
    (dict(dh=12), -2, "multiple of 8"), (dict(dh=136), -2, "multiple of 8"), (dict(dh=0), -1, "channels per head"),
    (dict(W=0), -1, "window"), (dict(S=-1), -1, "sinks"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=math.nan), -1, "scale"), (dict(scale=math.inf), -1, "scale"),
    (dict(n=-1), -1, "signal size"), (dict(n=1 << 31), -1, "signal size"), (dict(n=1 << 20, B=1 << 12), -2, "2^31"),
    (dict(q=None), -1, "q is NULL"), (dict(v=None), -1, "v is NULL"), (dict(y=None), -1, "y is NULL"),
    (dict(q=ODD), -1, "16-byte"), (dict(k_row=132), -1, "16-byte"), (dict(k_row=120), -1, "strides"),
    (dict(v_batch=-8), -1, "strides"), (dict(v_batch=4), -1, "16-byte"),
])
def test_sliding_refusals(L, args, code, fragment):
    expect(L, fwd(L, **args), code, fragment)


def test_sliding_nothing_to_do(L):
    assert fwd(L, n=0, q=None, k=None, v=None, y=None) == 0
    assert fwd(L, B=0, q=None) == 0


def bwd(L, work=P, wbytes=1 << 40, dk=P, dv=P, lse=P, dy=P, dy_row=256, dq=P, rest=None):
    return L.lib.circatt_sliding_bwd(3, 64, 2, 4, 2, 64, 16, 0, 0.125, P, 256, 0, P, 128, 0, P, 128, 0, None, P, rest, lse, dy,
                                     dy_row, 0, dq, dk, dv, work, wbytes, None)


@pytest.mark.parametrize("args,fragment", [
    (dict(work=None), "workspace is NULL"), (dict(wbytes=16), "workspace of 16"), (dict(work=ODD), "16-byte"),
    (dict(dk=None), "go together"), (dict(dv=None), "go together"), (dict(lse=None), "lse is NULL"),
    (dict(dy=None), "dy is NULL"), (dict(dy_row=8), "strides"), (dict(dq=None), "dq is NULL"),
])
def test_sliding_bwd_refusals(L, args, fragment):
    expect(L, bwd(L, **args), -1, fragment)


def test_workspace_sizes(L):
    w = L.lib.circatt_sliding_bwd_workspace_bytes
    assert w(3, 64, 2, 4, 2, 64, 16, 0) >= 4 * 64 * 2 * 4
    assert w(3, 0, 2, 4, 2, 64, 16, 0) == 0
    assert w(3, 64, 2, 4, 3, 64, 16, 0) == -1
    p = L.lib.circatt_paged_workspace_bytes
    assert p(3, 4, 4, 4, 2, 64, 16, 0, 16, 8) >= 0
    assert p(3, 0, 4, 4, 2, 64, 16, 0, 16, 8) == 0
    assert p(3, 4, 4, 4, 2, 60, 16, 0, 16, 8) == -1


def paged(L, dtype=3, T=4, B=4, H=4, Hk=2, dh=64, W=16, S=0, scale=0.125, q=P, q_row=256, ck=P, cv=P, npages=10, page=16,
          page_stride=2048, row_stride=128, pages=P, pages_row=8, maxp=8, lengths=P, offsets=None, y=P, work=P,
          wbytes=1 << 40):
    return L.lib.circatt_paged_attention(dtype, T, B, H, Hk, dh, W, S, scale, q, q_row, ck, cv, npages, page, page_stride,
                                         row_stride, pages, pages_row, maxp, lengths, offsets, y, 1, work, wbytes, None)


@pytest.mark.parametrize("args,code,fragment", [
    (dict(dtype=1), -2, "dtype"), (dict(dh=20), -2, "multiple of 8"), (dict(W=0), -1, "window"),
    (dict(page=24), -2, "power of two"), (dict(page=1 << 17), -2, "power of two"), (dict(npages=0), -1, "pages"),
    (dict(npages=1 << 40), -1, "pages"), (dict(maxp=0), -1, "page table"), (dict(pages_row=4), -1, "page table"),
    (dict(maxp=1 << 28, pages_row=1 << 28), -1, "page table"), (dict(pages=None), -1, "pages is NULL"),
    (dict(lengths=None), -1, "lengths is NULL"), (dict(row_stride=64), -1, "cache strides"),
    (dict(row_stride=132), -1, "16-byte"), (dict(ck=ODD), -1, "16-byte"), (dict(cv=None), -1, "cache is NULL"),
    (dict(T=5), -1, "without offsets"), (dict(q=None), -1, "q is NULL"), (dict(y=ODD), -1, "16-byte"),
    (dict(B=0), -1, "sizes"), (dict(T=-1, offsets=P), -1, "sizes"),
    (dict(npages=1 << 24, page_stride=1 << 12), -2, "63 GiB"), (dict(npages=1, row_stride=1 << 25), -2, "63 GiB"),
])
def test_paged_refusals(L, args, code, fragment):
    expect(L, paged(L, **args), code, fragment)


def test_paged_nothing_to_do(L):
    assert paged(L, T=0, offsets=P, q=None, y=None, work=None, wbytes=0) == 0


def append(L, dtype=3, T=4, B=4, C=128, k=P, k_row=128, v=P, v_row=128, ck=P, cv=P, npages=10, page=16, page_stride=2048,
           row_stride=128, pages=P, pages_row=8, maxp=8, lengths=P, offsets=None):
    return L.lib.circatt_paged_append(dtype, T, B, C, k, k_row, v, v_row, ck, cv, npages, page, page_stride, row_stride,
                                      pages, pages_row, maxp, lengths, offsets, None)


@pytest.mark.parametrize("args,code,fragment", [
    (dict(dtype=5), -2, "dtype"), (dict(T=-1), -1, "token count"), (dict(C=0), -1, "channel count"),
    (dict(page=3), -2, "power of two"), (dict(B=0), -1, "sequence count"), (dict(T=3), -1, "without offsets"),
    (dict(k=None), -1, "k is NULL"), (dict(v_row=-1), -1, "negative stride"), (dict(page_stride=64), -1, "cache strides"),
])
def test_append_refusals(L, args, code, fragment):
    expect(L, append(L, **args), code, fragment)


def rotary(L, dtype=3, naxes=2, n=(8, 8, 1), tokens=64, nb=2, H=4, dh=64, p=(16, 16, 0), base=1e4, x=P, x_row=256,
           positions=None, pos_batch=0, y=ctypes.c_void_p(0x20000)):
    return L.lib.circatt_axial_rotary(dtype, 0, 0, naxes, *n, tokens, nb, H, dh, *p, base, x, x_row, positions, pos_batch,
                                      y, None)


@pytest.mark.parametrize("args,code,fragment", [
    (dict(dtype=1), -2, "dtype"), (dict(naxes=0), -1, "naxes"), (dict(naxes=4), -1, "naxes"),
    (dict(dh=63), -1, "heads"), (dict(H=0), -1, "heads"), (dict(p=(16, 0, 0)), -1, "pairs"),
    (dict(p=(16, 17, 0)), -1, "do not fit"), (dict(dh=512, x_row=2048, p=(100, 100, 0)), -2, "at most 128"),
    (dict(base=0.0), -1, "base"), (dict(base=math.nan), -1, "base"), (dict(tokens=65), -1, "grid of 64"),
    (dict(n=(1 << 20, 1 << 20, 1)), -1, "grid"), (dict(positions=P, pos_batch=100), -1, "positions"),
    (dict(x=None), -1, "x is NULL"), (dict(x_row=128), -1, "token stride"), (dict(y=P), -1, "alias"),
    (dict(tokens=-1, positions=P), -1, "sizes"), (dict(H=1 << 16, dh=1 << 10), -1, "heads"),
])
def test_rotary_refusals(L, args, code, fragment):
    expect(L, rotary(L, **args), code, fragment)


def test_rotary_nothing_to_do(L):
    assert rotary(L, nb=0, x=None, y=None) == 0
    assert rotary(L, n=(0, 8, 1), tokens=0, x=None, y=None) == 0


def test_python_layer_refuses():
    import circulant_attention as ca
    x = torch.zeros(1, 4, 32)
    with pytest.raises(ValueError, match="HIP device"):
        ca.sliding_mh_attention(x, x, x, 3, 2)
    with pytest.raises(ValueError, match="HIP device"):
        ca.paged_mh_attention(x[0], x, x, x, x, 3, 2)
    with pytest.raises(ValueError, match="HIP device"):
        ca.paged_append_(x, x, x[0], x[0], x, x)
    with pytest.raises(ValueError, match="HIP device"):
        ca.axial_rotary(x, (4,), 2)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ca.axial_rotary([1.0], (4,), 2)
    with pytest.raises(AssertionError, match="divisible"):
        ca.SlidingAttBlock(32, 8, 3)
    with pytest.raises(AssertionError, match="kv_heads"):
        ca.SlidingAttBlock(32, 8, 4, 3)


def test_the_restatement_gives_softmax_attention_and_its_gradients():
    """token_model against torch's autograd in 64 bits."""
    g = torch.Generator().manual_seed(0)
    B, n, H, Hk, D, W, S = 2, 23, 4, 2, 8, 6, 3
    q, k, v = (torch.randn(B, n, h * D, generator=g, dtype=torch.float64, requires_grad=True) for h in (H, Hk, Hk))
    dy = torch.randn(B, n, H * D, generator=g, dtype=torch.float64)
    see = M.visible(torch.arange(n), n, W, S)
    assert [int(t) for t in see.sum(1)] == [min(i + 1, W + S) for i in range(n)]
    kk, vv = (t.reshape(B, n, Hk, 1, D).expand(-1, -1, -1, H // Hk, -1).reshape(B, n, H, D).transpose(1, 2) for t in (k, v))
    s = (q.reshape(B, n, H, D).transpose(1, 2) @ kk.transpose(-1, -2)) * 0.3
    y = (s.masked_fill(~see, -math.inf).softmax(-1) @ vv).transpose(1, 2).reshape(B, n, H * D)
    want = [y, *torch.autograd.grad(y, (q, k, v), dy)]
    got = M.sliding(*(t.detach() for t in (q, k, v)), W, H, Hk, S, 0.3, None, torch.float32, dy)
    for (x, bound), w in zip(got, want):
        assert torch.allclose(x, w, rtol=1e-10, atol=1e-12) and (bound >= 0).all()


@pytest.mark.parametrize("args,fragment", [
    (dict(rest=ODD), "16-byte"), (dict(rest=P), "must not overlap y"), (dict(dtype=0, rest=P), "16-bit types"),
])
def test_rounding_rest_refusals(L, args, fragment):
    expect(L, fwd(L, **args), -1, fragment)
    if "dtype" not in args:
        expect(L, bwd(L, **args), -1, fragment)


@pytest.mark.parametrize("at", [
    dict(q=0x10000), dict(q=0x10000 + 4 * 512 - 16), dict(q=0x10000 - 3 * 512 - 512 + 16),
    dict(ck=0x10000 - 32), dict(cv=0x10000 - 40944),
])
def test_paged_result_over_its_inputs(L, at):
    """y is 4 rows of 512 bytes at 0x10000, q the same, a cache 10 pages of 4096 (40960 bytes)."""
    far = dict(q=0x100000, ck=0x200000, cv=0x300000)
    args = {n: ctypes.c_void_p(a) for n, a in {**far, **at}.items()}
    expect(L, paged(L, y=P, **args), -1, "must not overlap")
