"""Token attention where inputs are not finite: rows and keys that products have
spoilt are formed again, those that are not finite anyway are not, and none of it
makes a call of another order of time."""
import math

import pytest
import torch

import token_model as M
from token_plan import walk_split

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def timed(call):
    """(result, milliseconds) of the second of two calls."""
    e0, e1 = torch.cuda.Event(True), torch.cuda.Event(True)
    for _ in range(2):
        e0.record()
        out = call()
        e1.record()
    torch.cuda.synchronize()
    return out, e0.elapsed_time(e1)


# name: what of dy is not finite
BAD_DY = {
    "all NaN": lambda dy: dy.fill_(math.nan),
    "all inf": lambda dy: dy.fill_(math.inf),
    "inf of both signs": lambda dy: dy.mul_(math.inf),
    "a channel": lambda dy: dy[..., 5::64].fill_(math.inf),
    "every tenth row": lambda dy: dy[:, ::10].mul_(math.inf),
    "one number": lambda dy: dy[:, 1000, 7].fill_(math.inf),
}


@pytest.mark.parametrize("bad", BAD_DY)
@pytest.mark.parametrize("W,B", [(512, 8), (512, 1), (None, 1)])
def test_overflowed_step_takes_no_other_time(ca, bad, W, B):
    """Gradients that came in as infinities or NaN over finite q, k and v, as in a
    step whose loss was scaled too far: every gradient that they reach is not finite,
    the others are, and the step takes 5 ms more at most than a good one of 0.3 to 1."""
    L, H, Hk, D = 4096, 8, 4, 64
    assert (walk_split(B, L, H, Hk, D, W, 0, torch.float16)[0] == 1) == (B == 8)
    q, k, v, dy = (randn(3 + i, B, L, h * D, dtype=torch.float16).cuda() for i, h in enumerate((H, Hk, Hk, H)))
    BAD_DY[bad](dy)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=Hk)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    (y, dq, dk, dv), ms = timed(step)
    assert torch.isfinite(y).all()
    rows = ~torch.isfinite(dy).reshape(B, L, Hk, H // Hk, D).all(-1)      # rows of dy by head
    assert torch.equal(~torch.isfinite(dq).reshape(B, L, Hk, H // Hk, D).any(-1), rows)
    # keys that such a row sees: dk whole, dv in the channels of it
    i = torch.arange(L, device="cuda")
    see = (i[None] <= i[:, None]) & (i[None] > i[:, None] - (W or L))      # row, key
    reached = (see.T.float() @ rows.any(-1).transpose(0, 1).reshape(L, -1).float() > 0).reshape(L, B, Hk).transpose(0, 1)
    assert torch.equal(~torch.isfinite(dk).reshape(B, L, Hk, D).any(-1), reached)
    assert torch.equal(torch.isfinite(dk).reshape(B, L, Hk, D).all(-1), ~reached)
    chan = (~torch.isfinite(dy)).reshape(B, L, Hk, H // Hk, D).any(3).transpose(0, 1).reshape(L, -1).float()
    chan = (see.T.float() @ chan > 0).reshape(L, B, Hk, D).transpose(0, 1)
    assert torch.equal(~torch.isfinite(dv).reshape(B, L, Hk, D), chan)
    assert ms < 6.0, ms


BAD_V = {
    "all NaN": lambda v: v.fill_(math.nan),
    "all inf": lambda v: v.fill_(math.inf),
    "a channel": lambda v: v[..., 5::64].fill_(math.nan),
    "every tenth row": lambda v: v[:, ::10].mul_(math.inf),
    "one number": lambda v: v[:, 1000, 7].fill_(math.inf),
}


@pytest.mark.parametrize("bad", BAD_V)
@pytest.mark.parametrize("W", [512, None])
def test_bad_values_take_no_other_time(ca, bad, W):
    """Values that are not finite under finite scores: the forward, and the same
    over a cache, in new tokens and in single ones."""
    L, H, Hk, D, page = 4096, 8, 4, 64, 64
    q, k, v = (randn(3 + i, 1, L, h * D, dtype=torch.float16).cuda() for i, h in enumerate((H, Hk, Hk)))
    BAD_V[bad](v)
    i = torch.arange(L, device="cuda")
    see = (i[None] <= i[:, None]) & (i[None] > i[:, None] - (W or L))
    chan = (see.float() @ (~torch.isfinite(v[0])).float() > 0).reshape(L, Hk, 1, D).expand(-1, -1, H // Hk, -1)
    want = chan.reshape(L, H * D)
    y, ms = timed(lambda: ca.sliding_mh_attention(q, k, v, W, H, kv_heads=Hk))
    assert torch.equal(~torch.isfinite(y[0]), want)
    assert ms < 6.0, ms
    cache = [t[0].reshape(L // page, page, Hk * D) for t in (k, v)]
    pages = torch.arange(L // page, dtype=torch.int32, device="cuda")[None]
    for new in (1, 700):
        offs = torch.tensor([0, new], dtype=torch.int32, device="cuda")
        lens = torch.full((1,), L, dtype=torch.int32, device="cuda")
        y, ms = timed(lambda: ca.paged_mh_attention(q[0, L - new:], *cache, pages, lens, W, H, kv_heads=Hk, offsets=offs))
        assert torch.equal(~torch.isfinite(y), want[L - new:]), new
        assert ms < 6.0, (new, ms)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(2, 200, 4, 2, 64, 30, 3), (1, 300, 6, 1, 128, 70, 50), (4, 512, 16, 16, 96, 64, 40)],
                         ids=str)
def test_what_single_numbers_do_not_reach_is_right(ca, shape, dtype):
    """Single numbers of v, or of dy, that are not finite: results that they do not
    reach, next to them in the products' tiles or in their own rows' other channels,
    are within the bounds of those without them."""
    B, L, H, Hk, D, W, S = shape
    dt = DT[dtype]
    assert (walk_split(*shape, dt)[0] == 1) == (B == 4)
    q, k, v, dy = (randn(23 + i, B, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H)))
    see = M.visible(torch.arange(L), L, W, S)
    tokens = (0, 5, S, 64, 65, 130, L - 1)

    def spoil(t):
        bad = torch.zeros(t.shape, dtype=torch.bool)
        for i, at in enumerate(tokens):
            bad[:, at, i * 11 % D::D] = True
        return torch.where(bad, torch.full((), math.inf if dtype == "f16" else math.nan, dtype=dt), t), bad

    def run(*args):
        leaves = [t.cuda().requires_grad_(True) for t in args[:3]]
        y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=Hk, sinks=S)
        return [t.cpu() for t in (y, *torch.autograd.grad(y, leaves, args[3].cuda()))]

    def reached(bad, sees):
        return (sees.float() @ bad.float().transpose(0, 1).reshape(L, -1) > 0).reshape(L, B, -1).transpose(0, 1)

    # values: y of the rows that see them, channel by channel
    spoilt, bad = spoil(v)
    y = run(q, k, spoilt, dy)[0]
    clean = torch.where(bad, torch.zeros_like(v), v)
    ((want, bound),) = M.sliding(*(t.double() for t in (q, k, clean)), W, H, Hk, S, 1 / math.sqrt(D), None, dt)
    hit = reached(bad, see).reshape(B, L, Hk, 1, D).expand(-1, -1, -1, H // Hk, -1).reshape(B, L, H * D)
    assert torch.equal(~torch.isfinite(y), hit)
    M.check(y[~hit], want[~hit], bound[~hit], "y")
    # rows of dy: dq of their own, dk of the keys that they see, dv in their channels
    spoilt, bad = spoil(dy)
    _, dq, dk, dv = run(q, k, v, spoilt)
    clean = torch.where(bad, torch.zeros_like(dy), dy)
    want = M.sliding(*(t.double() for t in (q, k, v)), W, H, Hk, S, 1 / math.sqrt(D), None, dt, clean.double())[1:]
    head = bad.reshape(B, L, H, D).any(-1, keepdim=True)
    hq = head.expand(-1, -1, -1, D).reshape(B, L, H * D)
    hk = reached(head.reshape(B, L, Hk, -1).any(-1), see.T).unsqueeze(-1).expand(-1, -1, -1, D).reshape(B, L, Hk * D)
    hv = reached(bad.reshape(B, L, Hk, H // Hk, D).any(3).reshape(B, L, -1), see.T)
    for got, (w, b), hit, name in zip((dq, dk, dv), want, (hq, hk, hv), ("dq", "dk", "dv")):
        assert torch.equal(~torch.isfinite(got), hit), name
        M.check(got[~hit], w[~hit], b[~hit], name)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("W,S", [(None, 0), (20, 3)])
def test_scores_of_minus_infinity_alone_give_nan(ca, dtype, W, S):
    """A row whose every visible score is -inf has no softmax: it is NaN, and so are
    the gradients of what it sees.  Over a cache as well, where a row that sees no
    token is zero."""
    L, H, Hk, D, page, t = 90, 4, 2, 32, 8, 60
    dt = DT[dtype]
    q, k, v, dy = (randn(53 + i, 1, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H)))
    k[..., ::D] = k[..., ::D].abs() + 1
    good = M.sliding(*(x.double() for x in (q, k, v)), W or L, H, Hk, S, 1 / math.sqrt(D), None, dt, dy.double())
    q[0, t] = 0
    q[0, t, ::D] = torch.tensor([1, -math.inf, 1, 1]).to(dt)
    leaves = [x.cuda().requires_grad_(True) for x in (q, k, v)]
    y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=Hk, sinks=S)
    _, dk, dv = (x.cpu()[0] for x in torch.autograd.grad(y, leaves, dy.cuda()))
    bad = torch.zeros(1, L, H * D, dtype=torch.bool)
    bad[0, t, D:2 * D] = True
    assert torch.equal(torch.isnan(y).cpu(), bad)
    other = torch.ones(L, dtype=torch.bool)
    other[t] = False
    M.check(y[:, other], good[0][0][:, other], good[0][1][:, other], "y")
    seen = M.visible(torch.arange(L), L, W or L, S)[t]
    for x in (dk, dv):
        assert torch.equal(torch.isnan(x).reshape(L, Hk, D)[..., 1:].all(-1)[:, 0], seen)
        assert torch.isfinite(x.reshape(L, Hk, D)[:, 1]).all() and torch.isfinite(x[~seen]).all()
    # the same tokens over a cache, where a second sequence's pages are not there and a
    # third one has no token
    caches = [torch.cat([x[0], torch.zeros(96 - L, Hk * D, dtype=dt)]).reshape(12, page, Hk * D).cuda() for x in (k, v)]
    for new in (40, 1):
        one = torch.arange(12, dtype=torch.int32)
        pages = torch.stack([one, torch.full_like(one, -1), one]).cuda()
        rows = q[0, t + 1 - new:t + 1]
        lens = torch.tensor([t + 1, t + 1, 0], dtype=torch.int32).cuda()
        offs = torch.tensor([0, new, 2 * new, 3 * new], dtype=torch.int32).cuda()
        got = ca.paged_mh_attention(rows.repeat(3, 1).cuda(), *caches, pages, lens, W, H, kv_heads=Hk, sinks=S, offsets=offs)
        assert (got[new:] == 0).all()
        assert torch.equal(torch.isnan(got[:new]).cpu(), bad[0, t + 1 - new:t + 1])
        if new > 1:
            M.check(got[:new - 1], good[0][0][0, t + 1 - new:t], good[0][1][0, t + 1 - new:t], "paged")
