"""The token operators' calls: what autograd and the arguments ask of them."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import token_model as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def test_tangents_are_refused_and_not_dropped(ca):
    """There is no forward mode: a tensor with a tangent is an error, also where no
    gradient is asked for, and others pass."""
    q = randn(1, 1, 20, 64).cuda()
    calls = (lambda x: ca.sliding_mh_attention(x, q, q, 5, 2), lambda x: ca.sliding_mh_attention(q, q, x, 5, 2),
             lambda x: ca.axial_rotary(x, (16,), 2))
    want = [f(q) for f in calls]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for f, w in zip(calls, want):
            with pytest.raises(RuntimeError, match="jvp"):
                f(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                f(dual)
            assert torch.equal(f(q), w)


@pytest.mark.parametrize("base", [12345.678, 10000 * 8 ** (64 / 62), 1.0e6 / 3, 2.5e8 + 1 / 3])
def test_rotary_base_that_float32_does_not_hold(ca, base):
    """The angle is formed in 64 bits from the base as it is given: within the
    restatement's bound (2^-21 of the pair's size, and rounding) to far positions,
    where the base rounded to Float32 is off by 1e-4 to 1e-3."""
    pos = torch.tensor([[0], [1], [-7], [1000], [100003], [1 << 20], [-(1 << 24) - 1]], dtype=torch.int32)
    x = randn(83, 7, 2 * 64)
    for interleaved in (False, True):
        t = x.cuda().requires_grad_(True)
        y = ca.axial_rotary(t, (32,), 2, positions=pos.cuda(), base=base, interleaved=interleaved)
        M.check(y, *M.rotary(x.double(), (32,), 2, base, pos, interleaved, torch.float32), "y")
        (g,) = torch.autograd.grad(y, t, x.cuda())
        M.check(g, *M.rotary(x.double(), (32,), 2, base, pos, interleaved, torch.float32, inverse=True), "dx")


def test_autograd_sees_what_is_written_in_place(ca):
    """A cache, or an `out`, that a graph has saved and a call then changes: the
    backward of that graph is an error, not a gradient of other values."""
    page, C, H = 8, 32, 2
    pages = torch.arange(4, dtype=torch.int32, device="cuda").reshape(2, 2)
    lens = torch.tensor([3, 9], dtype=torch.int32, device="cuda")
    new = randn(1, 2, C).cuda()
    caches = [randn(2 + i, 4, page, C).cuda() for i in range(2)]
    out = torch.zeros(2, C, device="cuda")
    before = [t._version for t in (*caches, out)]
    w = torch.ones(C, device="cuda", requires_grad=True)
    lost = [(t * w).sum() for t in (*caches, out)]
    kept = (new * w).sum()
    ca.paged_append_(*caches, new, new, pages, lens)
    ca.paged_mh_attention(new, *caches, pages, lens, None, H, out=out)
    assert all(t._version > n for t, n in zip((*caches, out), before))
    for loss in lost:
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    kept.backward()
    assert torch.equal(w.grad, new.sum(0))
    # views count with their base; tensors of inference mode have no counter
    both = torch.zeros(4, page, 2 * C, device="cuda")
    ca.paged_append_(*both.chunk(2, -1), new, new, pages, lens)
    assert both._version > 0
    with torch.inference_mode():
        frozen = [torch.zeros(4, page, C, device="cuda") for _ in range(2)]
        ca.paged_append_(*frozen, new, new, pages, lens)
        ca.paged_mh_attention(new, *frozen, pages, lens, None, H, out=torch.zeros(2, C, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offsets", [(0, 100, 5, 50), (0, 130, 2, 2), (0, 0, 150, 10), (90, 10, 0, 150), (0, -3, 70, 150),
                                     (0, 50, 1000, 1001), (5, 1 << 30, 7, 150), (-5, 3, 2, 1), (150, 0, 0, 0)])
def test_offsets_that_do_not_ascend_stay_inside(ca, dtype, offsets):
    """Offsets are documented to ascend from 0.  Others give unspecified rows, but
    nothing outside of the arrays is written, whatever they hold."""
    T, H, Hk, D, page, guard = 150, 4, 1, 32, 8, 300
    q = randn(1, T, H * D, dtype=dtype).cuda()
    caches = [randn(2 + i, 60, page, Hk * D, dtype=dtype).cuda() for i in range(2)]
    pages = torch.arange(60, dtype=torch.int32).reshape(3, 20).cuda()
    lens = torch.tensor([150, 140, 130], dtype=torch.int32).cuda()
    offs = torch.tensor(offsets, dtype=torch.int32).cuda()
    whole = torch.full((T + 2 * guard, H * D), 7.0, dtype=dtype, device="cuda")
    for W in (None, 9):
        ca.paged_mh_attention(q, *caches, pages, lens, W, H, kv_heads=Hk, sinks=2, offsets=offs, out=whole[guard:guard + T])
        ca.paged_mh_attention(q, *caches, pages, lens, W, H, kv_heads=Hk, sinks=2, offsets=offs)
        assert (whole[:guard] == 7).all() and (whole[guard + T:] == 7).all()
    kv = torch.full((62, page, Hk * D), 7.0, dtype=dtype, device="cuda")
    new = randn(4, T, Hk * D, dtype=dtype).cuda()
    ca.paged_append_(kv[1:61], kv[1:61].clone(), new, new, pages, lens, offsets=offs)
    assert (kv[0] == 7).all() and (kv[61] == 7).all()


def test_numbers_beyond_the_c_types(ca):
    """Windows and sinks of more than 64 bits hold every token; numbers of pairs of
    more than 32 are refused: none loses its high bits."""
    q = randn(1, 1, 40, 64).cuda()
    want = ca.sliding_mh_attention(q, q, q, None, 2)
    for big in ((1 << 64) + 5, (1 << 63) + 5):
        assert torch.equal(ca.sliding_mh_attention(q, q, q, big, 2), want)
        assert torch.equal(ca.sliding_mh_attention(q, q, q, 3, 2, sinks=big), want)
    for p in ((1 << 32) + 4, (1 << 64) + 4, -4, -(1 << 32) + 4):
        with pytest.raises(AssertionError, match="pairs"):
            ca.axial_rotary(q, (p,), 2)
