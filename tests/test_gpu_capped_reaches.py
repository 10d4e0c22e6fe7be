"""Equal products have equal capped scores, whatever else their tile holds: a tile's largest
product chooses the form of the tangent, and where the cap is large the forms' errors are
errors of the score that a softmax sees.

All keys that a row sees have the same product with it, so their weights are equal and the
softmax's reference is the one score: with f = 2^-24, u half a step of the type,
  y    u for a weight's rounding, u for the result's, (n + 16) f for sums, exponential, division
  dv   u, u, (n + 16) f likewise, and 2 f |lse| of the stored logarithm, which is a score's size
and, up to a cap of 256, the difference of two forms, 2^-21.5 + 2^-22 of the cap."""
import math

import pytest
import torch

from token_model import HALF, TINY

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
F = 2.0 ** -24


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def forms(cap):
    return cap * (2.0 ** -21.5 + 2.0 ** -22) if cap <= 256 else 256 * (2.0 ** -21.5 + 2.0 ** -22)


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("cap", [20.0, 256.0, 1000.0, 1e4, 1e5])
@pytest.mark.parametrize("reach,hidden", [(0.1, 0.5), (0.16, 0.5), (0.26, 0.9), (0.34, 0.9), (0.5, 1.2), (0.65, 3.0)])
def test_hidden_keys_leave_scores_alone(ca, dtype, cap, reach, hidden):
    """A first document's keys, hidden from the second's rows, lie in the second's first tile."""
    dt, n, first, D = DT[dtype], 200, 20, 32
    size = 64.0
    k = torch.zeros(n, D, dtype=dt)
    k[:, 0] = reach * size
    k[:first, 0] = hidden * size
    q = torch.zeros(n, D, dtype=dt)
    q[:, 0] = 1.0
    g = torch.Generator().manual_seed(1)
    v = torch.randn(n, D, generator=g).to(dt)
    v[:64, 0], v[64:, 0] = 1.0, -1.0
    dy = torch.randn(n, D, generator=g).to(dt)
    places = torch.tensor([list(range(first)) + list(range(n - first))], dtype=torch.int32, device="cuda")
    leaves = [t[None].cuda().requires_grad_(True) for t in (q, k, v)]
    y = ca.sliding_mh_attention(*leaves, n, 1, scale=cap / size, cap=cap, places=places)
    _, _, dv = torch.autograd.grad(y, leaves, dy[None].cuda())
    i = torch.arange(n)
    see = (i[None] <= i[:, None]) & ((i[None] < first) == (i[:, None] < first))
    p = see.double() / see.sum(1, keepdim=True)
    x = cap / size * (q.double() @ k.double().T).diagonal()
    lse = cap * torch.tanh(x / cap) + see.sum(1).double().log()
    u, tiny, v, dy, e = HALF[dt], TINY[dt], v.double(), dy.double(), (n + 16) * F + forms(cap)
    want, bound = p @ v, (u + e) * (p @ v.abs()) + u * (p @ v).abs() + tiny
    over = (y[0].detach().cpu().double() - want).abs() - bound
    assert over.max() <= 0, f"y: {over.max()} above its bound"
    w = p.T @ dy
    bound = (p * (u + e + 2 * F * lse.abs()[:, None])).T @ dy.abs() + u * w.abs() + tiny
    over = (dv[0].cpu().double() - w).abs() - bound
    assert over.max() <= 0, f"dv: {over.max()} above its bound"


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("cap", [20.0, 256.0, 1000.0, 1e4, 1e5])
@pytest.mark.parametrize("reach", [0.1, 0.16, 0.26, 0.5, 0.65])
def test_other_heads_leave_scores_alone(ca, dtype, cap, reach):
    """Over a paged cache two heads of queries share keys, and the second's products are large
    in the first half of the cache."""
    dt, n, D, page = DT[dtype], 256, 32, 16
    size = 64.0
    k = torch.zeros(n, D, dtype=dt)
    k[:, 0] = reach * size
    k[:n // 2, 1] = 0.9 * size
    q = torch.zeros(2, D, dtype=dt)
    q[0, 0] = q[1, 1] = 1.0
    v = torch.randn(n, D, generator=torch.Generator().manual_seed(1)).to(dt)
    v[:n // 2, 0], v[n // 2:, 0] = 1.0, -1.0
    cache = [t.reshape(n // page, page, D).cuda() for t in (k, v)]
    pages = torch.arange(n // page, dtype=torch.int32, device="cuda")[None]
    y = ca.paged_mh_attention(q.reshape(1, 2 * D).cuda(), *cache, pages, torch.tensor([n], dtype=torch.int32, device="cuda"), n, 2,
                              kv_heads=1, scale=cap / size, cap=cap)
    u, v = HALF[dt], v.double()
    want = v.mean(0)
    bound = (u + (n + 16) * F + forms(cap)) * v.abs().mean(0) + u * want.abs() + TINY[dt]
    over = (y[0, :D].cpu().double() - want).abs() - bound
    assert over.max() <= 0, f"{over.max()} above its bound"
