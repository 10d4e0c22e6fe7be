"""Single numbers that are not finite at drawn places of drawn shapes: what they do
not reach is within the 64-bit restatement's bounds of the inputs without them, and
what they reach is not finite."""
import math
import random

import pytest
import torch

import token_model as M
from token_plan import walk_split

pytestmark = pytest.mark.gpu
DT = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def spread(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def spoil(rng, t, rows):
    """(t with some numbers of the given rows not finite, where)"""
    bad = torch.zeros(t.shape, dtype=torch.bool)
    for i in rows:
        for _ in range(rng.choice([1, 1, 3])):
            bad[i, rng.randrange(t.shape[1])] = True
    value = rng.choice([math.nan, math.inf, -math.inf])
    return torch.where(bad, torch.full((), value, dtype=t.dtype), t), bad


def some(rng, n):
    return {rng.randrange(n) for _ in range(rng.choice([1, 2, 5]))} | ({n - 1} if rng.random() < 0.3 else set())


@pytest.mark.parametrize("seed", range(30))
def test_sliding(ca, seed):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    dt = DT[seed % 3]
    Hk, G, D = spread(rng, 1, 6), spread(rng, 1, 6), 8 * rng.randint(1, 16)
    H = Hk * G
    L, B = max(2, min(spread(rng, 2, 900), 60000 // H)), 1 if seed % 2 else 256 // Hk
    W, S = rng.choice([None, spread(rng, 1, 300)]), rng.choice([0, spread(rng, 1, 150)])
    if B > 1:
        L = min(L, 200)
    print("sliding", seed, dt, B, L, H, Hk, D, W, S, walk_split(B, L, H, Hk, D, W, S, dt)[:3], flush=True)
    q, k, v, dy = ([torch.randn(L, h * D, generator=g).to(dt) for h in (H, Hk, Hk, H)])
    n = rng.choice([L, rng.randint(1, L)])
    see = M.visible(torch.arange(n), n, W or L, S)
    lens = torch.full((B,), n, dtype=torch.int32).cuda()

    def run(*args):  # the same signal in every place of the batch, whose results are the same
        leaves = [t.cuda().expand(B, -1, -1).contiguous().requires_grad_(True) for t in args[:3]]
        y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=Hk, sinks=S, lengths=lens)
        out = [y, *torch.autograd.grad(y, leaves, args[3].cuda().expand(B, -1, -1).contiguous())]
        assert all(torch.equal(t[0].nan_to_num(1.5), t[-1].nan_to_num(1.5)) for t in out)
        return [t[0].detach().cpu() for t in out]

    def want(*args):
        return [(x[0, :n], b[0, :n]) for x, b in
                M.sliding(*(t[None].double() for t in args[:3]), W or L, H, Hk, S, 1 / math.sqrt(D), torch.tensor([n]), dt,
                          args[3][None].double())]

    def reached(bad, sees):
        return sees.float() @ bad[:n].float() > 0

    def compare(got, expect, hit, name):
        x, b = expect
        assert (got[n:] == 0).all(), name
        assert torch.equal(~torch.isfinite(got[:n]), hit), name
        M.check(got[:n][~hit], x[~hit], b[~hit], name)

    def wide(bad, heads):  # a head's flag to its channels
        return bad[:, :, None].expand(-1, -1, D).reshape(bad.shape[0], heads * D)

    # a value: the rows that see it, in its channel
    t, bad = spoil(rng, v, some(rng, n))
    hit = reached(bad, see).reshape(n, Hk, 1, D).expand(-1, -1, G, -1).reshape(n, H * D)
    compare(run(q, k, t, dy)[0], want(q, k, torch.where(bad, torch.zeros_like(v), v), dy)[0], hit, "y")
    # a row of dy: its dq, dk of the keys that it sees, dv in its channels
    t, bad = spoil(rng, dy, some(rng, n))
    got, expect = run(q, k, v, t)[1:], want(q, k, v, torch.where(bad, torch.zeros_like(dy), dy))[1:]
    head = bad[:n].reshape(n, H, D).any(-1)
    compare(got[0], expect[0], wide(head, H), "dq")
    compare(got[1], expect[1], wide(reached(head.reshape(n, Hk, G).any(-1), see.T), Hk), "dk")
    compare(got[2], expect[2], reached(bad[:n].reshape(n, Hk, G, D).any(2).reshape(n, -1), see.T), "dv")
    # a query of NaN: its y and dq, and the gradients of what it sees
    at = sorted(some(rng, n))
    t = q.clone()
    t[at] = math.nan
    zero = q.clone()
    zero[at] = 0
    gone = dy.clone()
    gone[at] = 0
    got, expect = run(t, k, v, dy), want(zero, k, v, gone)
    rows = torch.zeros(n, dtype=torch.bool)
    rows[at] = True
    keys = reached(rows[:, None], see.T)[:, 0]
    for x, e, r, name in zip(got[:2], expect[:2], (rows, rows), ("y", "dq")):
        # (y of the others does not hang on dy, dq of them not on the rows left out)
        compare(x, e, r[:, None].expand(-1, H * D), name)
    for x, e, name in zip(got[2:], expect[2:], ("dk", "dv")):
        compare(x, e, keys[:, None].expand(-1, Hk * D), name)


@pytest.mark.parametrize("seed", range(30))
def test_paged(ca, seed):
    rng, g = random.Random(500 + seed), torch.Generator().manual_seed(seed)
    dt = DT[seed % 3]
    Hk, G, D, page = spread(rng, 1, 6), spread(rng, 1, 8), 8 * rng.randint(1, 16), 2 ** rng.randint(0, 7)
    H, B = Hk * G, rng.choice([1, 3, 40])
    seqs = [(n, m if seed % 2 else 1) for n, m in ((spread(rng, 2, 1200 if B < 40 else 200), 0) for _ in range(B))
            for m in [min(n, spread(rng, 1, 150))]]
    need = [-(-n // page) for n, _ in seqs]
    pages = torch.full((B, max(need) + 1), -1, dtype=torch.int32)
    order = torch.randperm(sum(need), generator=g).to(torch.int32)
    at = 0
    for b, n in enumerate(need):
        pages[b, :n] = order[at:at + n]
        at += n
    k, v = (torch.randn(sum(need), page, Hk * D, generator=g).to(dt) for _ in range(2))
    lens = torch.tensor([n for n, _ in seqs], dtype=torch.int32)
    offs = torch.tensor([0] + [m for _, m in seqs], dtype=torch.int32).cumsum(0).to(torch.int32)
    q = torch.randn(int(offs[-1]), H * D, generator=g).to(dt)
    W, S = rng.choice([None, spread(rng, 1, 300)]), rng.choice([0, spread(rng, 1, 150)])
    print("paged", seed, dt, "H", H, Hk, D, "page", page, "W", W, S, seqs[:4], B, flush=True)
    hit = torch.zeros(q.shape[0], Hk, D, dtype=torch.bool)
    spoilt, clean = v.clone(), v.clone()
    for b in range(0, B, 2):
        n, m = seqs[b]
        lo = int(offs[b])
        for j in some(rng, n):
            slot, c = (int(pages[b, j // page]), j % page), rng.randrange(Hk * D)
            spoilt[slot][c], clean[slot][c] = rng.choice([math.nan, math.inf]), 0
            hit[lo:lo + m, c // D, c % D] |= M.visible(torch.arange(n - m, n), n, W or 1 << 30, S)[:, j]
    hit = hit[:, :, None].expand(-1, -1, G, -1).reshape(q.shape[0], H * D)
    want, bound = M.paged(q.double(), k.double(), clean.double(), pages, lens, offs, W or 1 << 30, H, Hk, S, 1 / math.sqrt(D),
                          dt)
    y = ca.paged_mh_attention(*(t.cuda() for t in (q, k, spoilt, pages, lens)), W, H, kv_heads=Hk, sinks=S,
                              offsets=offs.cuda()).cpu()
    assert torch.equal(~torch.isfinite(y), hit)
    M.check(y[~hit], want[~hit], bound[~hit], "y")
