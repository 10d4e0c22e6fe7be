"""Gradients of capped scores far into saturation, relative to what they are, against 64 bits.

The derivative of cap tanh(x / cap) is 1 - t^2 = 4 r (1 - r), r = 1 / (1 + E), E = exp(2 |x| / cap).
From E's relative error e it is off by t e <= e of itself, from the reciprocal and the sum in
it by 2^-23 + 2^-24 (of r, less of 1 - r), by one rounding of the product, and E's own error is
2^-23 of the exponential, the two roundings of its exponent z = 2 log2(e) |x| / cap, 2 f z ln 2
(f = 2^-24), and 2 / cap times x's.  Where a series gives t instead (|x| / cap <= 0.7), t <= 0.61
and its error of 2^-21 of the cap leave 1 - t^2 >= 0.63 off by 2^-20.9.  In all
    2^-20 + 2 ln 2 f z + 2 error(x) / cap   of the derivative.
The products of these inputs are sums of few small whole numbers times powers of two, exact in
Float32, so that x is off by the one rounding of the scale in it: f |x|."""
import math

import pytest
import torch

from token_model import HALF, TINY

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F = 2.0 ** -24


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def reference(q, k, v, dy, see, scale, cap, dtype):
    """[(value, bound)] of dq, dk of one head in 64 bits; rows of k, v that nobody sees take
    no part."""
    u, tiny = HALF[dtype], TINY[dtype]
    n, D = k.shape
    used = see.any(0)[:, None]
    k, v = (torch.where(used, t, torch.zeros_like(t)) for t in (k, v))
    x = (q @ k.T) * scale
    z = 2 * math.log2(math.e) * x.abs() / cap
    bend = 1 / torch.cosh(x / cap) ** 2
    ebend = bend * (2.0 ** -20 + 2 * math.log(2) * F * z + 2 * F * x.abs() / cap)
    s = cap * torch.tanh(x / cap)
    es = cap * 2.0 ** -21 + F * x.abs() * bend + 2 * F * s.abs()
    s = s.masked_fill(~see, -math.inf)
    p = s.softmax(1)
    lse = torch.logsumexp(s, 1, keepdim=True).abs() * 2 * F
    e = es + (p * es).sum(1, keepdim=True) + (n + 16) * F + lse
    y = p @ v
    by = (p * (u + e)) @ v.abs() + u * y.abs() + tiny * (v.abs().sum(0) + 1)
    d = (dy * y).sum(1, keepdim=True)
    bd = ((u * y.abs() + by) * dy.abs()).sum(1, keepdim=True) + D * F * (dy * y).abs().sum(1, keepdim=True)
    ds = p * (dy @ v.T - d)
    bds = e * ds.abs() + p * (bd + (D + 3) * F * (dy.abs() @ v.abs().T))
    dx = ds * bend
    bdx = torch.where(see, u * dx.abs() + bds * (bend + ebend) + ds.abs() * ebend + tiny, torch.zeros_like(x))
    dq, dk = scale * (dx @ k), scale * (dx.T @ q)
    bdq = scale * (bdx @ k.abs()) + (u + n * F) * scale * (dx.abs() @ k.abs()) + tiny
    bdk = scale * (bdx.T @ q.abs()) + (u + n * F) * scale * (dx.abs().T @ q.abs()) + tiny
    return [(dq, bdq), (dk, bdk)]


def inputs(n, D, reach, cap, dtype, seed, sign=1.0):
    """Scores of some reach times the cap, few of them alike: x = 0.125 q k with q[0] = 8 reach
    cap (and k[0] = sign) and two small whole numbers more."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randint(-2, 3, (n, D), generator=g).double()
    q = torch.zeros(n, D).double()
    k[:, 0] = sign
    q[:, 0] = 8 * reach * cap
    q[:, 1:3] = torch.randint(-1, 2, (n, 2), generator=g).double()
    v = torch.randn(n, D, generator=g).to(dtype).double()
    dy = (torch.randn(n, D, generator=g) * 1024).to(dtype).double()  # (Float16 holds what the derivative leaves)
    return q, k, v, dy


def check(got, want, bound, what):
    got = got.cpu().double()
    over = ((got - want).abs() - bound).max().item()
    assert over <= 0, f"{what}: {over} above its bound"


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("reach", [0.25, 0.5, 1, 2, 4, 6, 7, 8, 9])
def test_gradients_of_saturated_scores(ca, dtype, reach):
    dt, cap, scale, D = DT[dtype], 2.0, 0.125, 32
    for n, W, sign in ((40, 40, 1.0), (300, 64, 1.0), (300, 300, -1.0)):
        q, k, v, dy = inputs(n, D, reach, cap, dt, 3 + n, sign)
        i = torch.arange(n)
        see = (i[None] <= i[:, None]) & (i[None] > i[:, None] - W)
        leaves = [t.to(dt)[None].cuda().requires_grad_(True) for t in (q, k, v)]
        y = ca.sliding_mh_attention(*leaves, W, 1, scale=scale, cap=cap)
        got = torch.autograd.grad(y, leaves, dy.to(dt)[None].cuda())
        for g, (w, b), name in zip(got, reference(q, k, v, dy, see, scale, cap, dt), ("dq", "dk")):
            check(g[0], w, b, f"{name}, {n} tokens, window {W}")


@pytest.mark.parametrize("dtype", sorted(DT))
def test_gradients_of_saturated_scores_formed_again(ca, dtype):
    """Rows whose tiles hold a token that is not finite and that they do not see, and keys whose
    rows' tiles do: row by row, with the same derivative."""
    dt, cap, scale, D, n, W, reach = DT[dtype], 2.0, 0.125, 32, 200, 20, 7
    q, k, v, dy = inputs(n, D, reach, cap, dt, 11)
    bad = 70
    i = torch.arange(n)
    see = (i[None] <= i[:, None]) & (i[None] > i[:, None] - W)
    reached = see[:, bad]                       # rows that see it, and the keys that those see
    keys = see[reached].any(0)
    k2 = k.clone()
    k2[bad, 5] = math.nan
    leaves = [t.to(dt)[None].cuda().requires_grad_(True) for t in (q, k2, v)]
    y = ca.sliding_mh_attention(*leaves, W, 1, scale=scale, cap=cap)
    dq, dk, _ = (t[0].cpu() for t in torch.autograd.grad(y, leaves, dy.to(dt)[None].cuda()))
    (wq, bq), (wk, bk) = reference(q, k, v, dy, see, scale, cap, dt)
    check(dq[~reached], wq[~reached], bq[~reached], "dq")
    check(dk[~keys], wk[~keys], bk[~keys], "dk")
    assert dq[reached].isnan().all() and dk[keys].isnan().any(1).all()
