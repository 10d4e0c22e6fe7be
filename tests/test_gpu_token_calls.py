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
