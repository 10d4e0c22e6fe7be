"""A serving step captured whole: fork, resize, append, attend and compact, by the forms of the
page operators that take one workgroup and by those that plan and apply, replayed with other
tables, lengths, sources and tokens, against lists and 64 bits."""
import random

import pytest
import torch

import pages_model as P
import shaped_model as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(r, B, most, page, npages):
    """(rows, lengths, counts): each sequence with its own pages, some without tokens."""
    order = list(range(npages))
    r.shuffle(order)
    rows, lengths, at = [], [], 0
    for _ in range(B):
        n = r.choice([0, r.randint(1, (most - 2) * page), r.randint(1, 2 * page)])
        has = -(-n // page)
        rows.append(order[at:at + has] + [-1] * (most - has))
        lengths.append(n)
        at += has
    assert at <= npages
    counts = [0] * npages
    for row in rows:
        for p in row:
            if p >= 0:
                counts[p] += 1
    return rows, lengths, counts


def held(rows, lengths, cache, page):
    """A sequence's tokens, by its row."""
    out = []
    for row, n in zip(rows, lengths):
        j = torch.arange(n)
        out.append(cache[torch.tensor(row, dtype=torch.long)[j // page], j % page] if n else cache[:0, 0])
    return out


@pytest.mark.parametrize("B,most,npages", [
    (6, 8, 60),           # one workgroup each
    (70, 40, 3200),       # a plan with the counts in LDS, and its work
    (5, 40, 33000),       # a plan with the counts in memory
    (1100, 8, 6000),      # (of more sequences than the plan's threads)
])
def test_a_step_captured_and_replayed(ca, B, most, npages):
    H, Hk, D, W, page, dt = 2, 1, 32, 24, 8, torch.bfloat16
    r, g = random.Random(B), torch.Generator().manual_seed(B)
    C = Hk * D
    k, v = (torch.zeros((npages, page, C), dtype=dt, device="cuda") for _ in range(2))
    args = [ints([[-1] * most] * B), ints([0] * B), ints([0] * npages), ints([0] * B), ints([0] * B), ints([0] * (B + 1))]
    pages, lengths, counts, source, to, offsets = args
    T = 2 * B
    q, kn, vn = (torch.zeros((T, h * D), dtype=dt, device="cuda") for h in (H, Hk, Hk))

    def step():
        forked = ca.paged_fork(pages, lengths, counts, source, page)
        grown = ca.paged_resize_(k, v, *forked, to)
        ca.paged_append_(k, v, kn, vn, grown[0], grown[1], offsets=offsets)
        y = ca.paged_mh_attention(q, k, v, grown[0], grown[1], W, H, kv_heads=Hk, sinks=1, offsets=offsets, cap=10.0)
        packed = ca.paged_compact_(k, v, grown[0], grown[2])
        return (*grown, y, *packed)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        rows, n0, c0 = pool(r, B, most, page, npages)
        src = [r.randrange(B) for _ in range(B)]
        f = P.fork(rows, n0, c0, src, page)
        want = [n + r.choice([1, 2, 1, 1]) if n < (most - 1) * page else -1 for n in f[1]]
        w = P.resize(*f, want, page)
        new = [b - a for a, b in zip(f[1], w[1])]
        offs = [0]
        for m in new:
            offs.append(offs[-1] + m)
        for t, x in zip(args, (rows, n0, c0, src, want, offs)):
            t.copy_(torch.tensor(x, dtype=torch.int32))
        tokens = [torch.randn((T, h * D), generator=g).to(dt) for h in (H, Hk, Hk)]
        before = [torch.randn((npages, page, C), generator=g).to(dt) for _ in range(2)]
        for t, x in zip((q, kn, vn, k, v), (*tokens, *before)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        z = P.compact(w[0], w[2])
        for got, x in zip((*out[:3], *out[4:]), (*w[:3], *z[:2])):
            assert got.cpu().tolist() == x
        # tokens of every sequence, where the pages lie in the end
        ends = []
        for cache, old, fresh in zip((k, v), before, tokens[1:]):
            was = held(f[0], f[1], old, page)
            now = held(z[0], w[1], cache.cpu(), page)
            for b in range(B):
                assert torch.equal(now[b], torch.cat([was[b], fresh[offs[b]:offs[b + 1]]])), f"sequence {b}"
            ends.append(cache.cpu().double())
        some = list(range(B)) if B <= 100 else r.sample(range(B), 100)
        qd = torch.cat([tokens[0][offs[b]:offs[b + 1]] for b in some]).double()
        so = [0]
        for b in some:
            so.append(so[-1] + new[b])
        x, bx = M.paged(qd, *ends, torch.tensor([z[0][b] for b in some]), torch.tensor([w[1][b] for b in some]),
                        torch.tensor(so), W, H, Hk, 1, D ** -0.5, dt, cap=10.0)
        y = torch.cat([out[3][offs[b]:offs[b + 1]] for b in some]).cpu()
        M.check(y, x, bx, "attention")
        assert not out[3][offs[-1]:].any()
