"""Token attention on shapes drawn from its whole range, against the 64-bit
restatement within its bounds: heads, groups, widths, windows, sinks, ragged
lengths, strides, pages, mixed batches, each element type."""
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


def randn(g, *shape, dtype):
    return torch.randn(shape, generator=g).to(dtype)


def spread(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


@pytest.mark.parametrize("seed", range(36))
def test_sliding(ca, seed):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    dt = DT[seed % 3]
    Hk, G, D, B = spread(rng, 1, 8), spread(rng, 1, 9), 8 * rng.randint(1, 16), spread(rng, 1, 8)
    H = Hk * G
    L = max(1, min(spread(rng, 1, 900), 150000 // (B * H)))
    W, S = rng.choice([None, spread(rng, 1, 400)]), rng.choice([0, spread(rng, 1, 200)])
    lens = None if rng.random() < 0.5 else torch.tensor([rng.randint(0, L) for _ in range(B)], dtype=torch.int32)
    print("sliding", seed, dt, B, L, H, Hk, D, W, S, lens, walk_split(B, L, H, Hk, D, W, S, dt)[:3], flush=True)
    gap = 8 * rng.randint(0, 3)
    qkv = randn(g, B, L, (H + 2 * Hk) * D + gap, dtype=dt)
    q, k, v = qkv[..., :(H + 2 * Hk) * D].split([H * D, Hk * D, Hk * D], -1)
    dy = randn(g, B, L, H * D, dtype=dt)
    whole = qkv.cuda().requires_grad_(True)
    y = ca.sliding_mh_attention(*whole[..., :(H + 2 * Hk) * D].split([H * D, Hk * D, Hk * D], -1), W, H, kv_heads=Hk, sinks=S,
                                lengths=None if lens is None else lens.cuda())
    (grad,) = torch.autograd.grad(y, whole, dy.cuda())
    want = M.sliding(*(t.double() for t in (q, k, v)), W or L, H, Hk, S, 1 / math.sqrt(D), lens, dt, dy.double())
    for got, (x, bx), name in zip((y, *grad[..., :(H + 2 * Hk) * D].split([H * D, Hk * D, Hk * D], -1)), want,
                                  ("y", "dq", "dk", "dv")):
        M.check(got, x, bx, name)


@pytest.mark.parametrize("seed", range(36))
def test_paged(ca, seed):
    rng, g = random.Random(100 + seed), torch.Generator().manual_seed(seed)
    dt = DT[seed % 3]
    Hk, G, D, page = spread(rng, 1, 8), spread(rng, 1, 9), 8 * rng.randint(1, 16), 2 ** rng.randint(0, 7)
    H, B = Hk * G, spread(rng, 1, 80)
    kind, most = seed % 4, 40000 // B
    seqs = []
    for _ in range(B):
        n = spread(rng, 1, min(most, 1500)) if rng.random() < 0.93 else 0
        m = 1 if kind == 0 else rng.choice([0, 1, 1, 2, min(n, 9)]) if kind == 1 else spread(rng, 1, max(n, 1))
        seqs.append((n, min(m, 200) if kind < 3 else rng.choice([1, min(m, 200)])))
    need = [-(-n // page) for n, _ in seqs]
    pages = torch.full((B, max(max(need), 1) + rng.randint(0, 3)), -1, dtype=torch.int32)
    order = torch.randperm(sum(need) + 2, generator=g).to(torch.int32)
    at = 0
    for b, n in enumerate(need):
        pages[b, :n] = order[at:at + n]
        at += n
        if n and rng.random() < 0.1:
            pages[b, rng.randrange(n)] = rng.choice([-1, 1 << 30])
    caches = [randn(g, sum(need) + 2, page, Hk * D, dtype=dt) for _ in range(2)]
    lens = torch.tensor([n for n, _ in seqs], dtype=torch.int32)
    offs = torch.tensor([0] + [m for _, m in seqs], dtype=torch.int32).cumsum(0).to(torch.int32)
    q = randn(g, int(offs[-1]) + rng.randint(0, 2), H * D, dtype=dt)
    W, S = rng.choice([None, spread(rng, 1, 400)]), rng.choice([0, spread(rng, 1, 200)])
    print("paged", seed, dt, "H", H, Hk, D, "page", page, "W", W, S, "B", B, "T", q.shape[0], flush=True)
    want, bound = M.paged(q.double(), *(t.double() for t in caches), pages, lens, offs, W or 1 << 30, H, Hk, S,
                          1 / math.sqrt(D), dt)
    y = ca.paged_mh_attention(*(t.cuda() for t in (q, *caches, pages, lens)), W, H, kv_heads=Hk, sinks=S, offsets=offs.cuda())
    M.check(y, want, bound, "y")
