"""paged_fork, paged_resize_ and paged_compact_ against pages_model.py, number by number and
byte by byte, and a serving loop over them against a cache of its own for each sequence."""
import math
import random

import pytest
import torch

import pages_model as P
import shaped_model as M

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def same(got, want):
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), torch.tensor(want, dtype=torch.int32).reshape(got.shape))


def pool(r, B, most, page, npages, outside=False, share=0.3):
    """Rows, lengths and counts of B sequences, some of which share their pages."""
    free, rows, lengths = list(range(npages)), [], []
    r.shuffle(free)
    counts = [0] * npages
    for b in range(B):
        if b and r.random() < share:
            rows.append(list(rows[-1]))
            lengths.append(lengths[-1])
        else:
            n = r.choice([0, 1, page, r.randint(0, most * page), r.randint(0, most * page)])
            n = min(n, len(free) * page)
            has = P.reach(n, page, most)
            rows.append([free.pop() for _ in range(has)] + [-1] * (most - has))
            if outside and has and r.random() < 0.3:
                at = r.randrange(has)
                free.append(rows[-1][at])
                rows[-1][at] = r.choice([-1, npages, 2 ** 31 - 1, -2 ** 31])
            lengths.append(n)
        for p in rows[-1][:P.reach(lengths[-1], page, most)]:
            if 0 <= p < npages:
                counts[p] += 1
    return rows, lengths, counts


SIZES = [(1, 1, 1, 1), (1, 3, 4, 7), (5, 7, 16, 30), (17, 9, 8, 200), (64, 33, 16, 1500), (300, 5, 2, 2000), (3, 700, 16, 40000),
         (1100, 4, 1, 5000)]


@pytest.mark.parametrize("outside", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_fork(ca, size, outside):
    B, most, page, npages = size
    r = random.Random(B + outside)
    rows, lengths, counts = pool(r, B, most, page, npages, outside)
    for N in (0, 1, B, 2 * B + 3):
        source = [r.choice([-1, B, 2 ** 31 - 1]) if r.random() < 0.1 else r.randrange(B) for _ in range(N)]
        got = ca.paged_fork(ints(rows), ints(lengths), ints(counts), ints(source), page)
        for g, w in zip(got, P.fork(rows, lengths, counts, source, page)):
            same(g, w)
    # lengths that pass the table, or lie below zero
    odd = [r.choice([-7, 2 ** 31 - 1, n]) for n in lengths]
    source = list(range(B))
    got = ca.paged_fork(ints(rows), ints(odd), ints(counts), ints(source), page)
    for g, w in zip(got, P.fork(rows, odd, counts, source, page)):
        same(g, w)


def caches(npages, page, C, dt, kind="plain"):
    g = torch.Generator(device="cuda").manual_seed(npages + C)
    if kind == "strided":  # k and v side by side, tokens apart
        both = torch.randn((npages, page, 2, C + 16), device="cuda", generator=g).to(dt)
        return both[:, :, 0, :C], both[:, :, 1, :C]
    return tuple(torch.randn((npages, page, C), device="cuda", generator=g).to(dt) for _ in range(2))


def moved(cache, moves, page):
    out = cache.clone()
    for a, b, *n in moves:
        out[b, :(n[0] if n else page)] = cache[a, :(n[0] if n else page)]
    return out


@pytest.mark.parametrize("dtype,C,kind", [("bf16", 64, "plain"), ("f16", 40, "strided"), ("f32", 24, "plain")])
@pytest.mark.parametrize("outside", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_resize(ca, size, outside, dtype, C, kind):
    B, most, page, npages = size
    r = random.Random(B + outside)
    rows, lengths, counts = pool(r, B, most, page, npages, outside, share=0.5)
    for _ in range(3):
        to = [r.choice([-1, 0, n, n + 1, n + r.randint(0, 3 * page), r.randint(0, max(n, 1)), 2 ** 31 - 1 if r.random() < 0.1 else n + 1])
              for n in lengths]
        k, v = caches(npages, page, C, DT[dtype], kind)
        k0, v0, version = k.clone(), v.clone(), (k._version, v._version)
        got = ca.paged_resize_(k, v, ints(rows), ints(lengths), ints(counts), ints(to))
        assert k._version > version[0] and v._version > version[1]
        *want, moves = P.resize(rows, lengths, counts, to, page)
        for g, w in zip(got, want):
            same(g, w)
        assert torch.equal(k, moved(k0, moves, page)) and torch.equal(v, moved(v0, moves, page))
        rows, lengths, counts = want


@pytest.mark.parametrize("dtype,C,kind", [("bf16", 64, "plain"), ("f16", 40, "strided"), ("f32", 24, "plain")])
@pytest.mark.parametrize("outside", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_compact(ca, size, outside, dtype, C, kind):
    B, most, page, npages = size
    r = random.Random(B + outside)
    rows, lengths, counts = pool(r, B, most, page, npages, outside)
    # half of the sequences end
    rows, lengths, counts, _ = P.resize(rows, lengths, counts, [r.choice([0, -1]) for _ in range(B)], page)
    k, v = caches(npages, page, C, DT[dtype], kind)
    k0, v0 = k.clone(), v.clone()
    got = ca.paged_compact_(k, v, ints(rows), ints(counts))
    *want, moves = P.compact(rows, counts)
    for g, w in zip(got, want):
        same(g, w)
    assert torch.equal(k, moved(k0, moves, page)) and torch.equal(v, moved(v0, moves, page))
    used = int((got[1] > 0).sum())
    assert (got[1][used:] <= 0).all() and (got[1][:used] > 0).all()


def test_too_few_pages(ca):
    """The first that finds too few and those behind it stay; one that needs none goes on,
    and what others give back in the call is given."""
    page, npages = 4, 8
    rows = [[0, 1, -1, -1], [2, -1, -1, -1], [3, 4, -1, -1], [5, -1, -1, -1], [6, -1, -1, -1]]
    lengths, counts = [8, 4, 7, 3, 4], [1] * 7 + [0]
    to = [0, 12, 8, 15, 5]  # gives 2; takes 2; needs none; needs 3, 1 is there; needs 1
    k, v = caches(npages, page, 16, torch.bfloat16)
    got = ca.paged_resize_(k, v, ints(rows), ints(lengths), ints(counts), ints(to))
    same(got[1], [0, 12, 8, 3, 4])
    *want, moves = P.resize(rows, lengths, counts, to, page)
    assert not moves
    for g, w in zip(got, want):
        same(g, w)


def test_serving_with_beams(ca):
    """Prompts, forks, single tokens, sequences that end, and a compaction, against a cache
    without pages for each sequence; every step captured once and replayed twice more."""
    H, Hk, D, page, npages, most, W, dt = 4, 2, 32, 8, 120, 12, 30, torch.bfloat16
    r, g = random.Random(4), torch.Generator().manual_seed(4)
    k, v = caches(npages, page, Hk * D, dt)
    B = 3
    pages, lengths, counts = ints([[-1] * most] * B), ints([0] * B), ints([0] * npages)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.05], device="cuda")
    kept = [[[], []] for _ in range(B)]

    def step(to):
        nonlocal pages, lengths, counts
        old = lengths.tolist()
        pages, lengths, counts = ca.paged_resize_(k, v, pages, lengths, counts, ints(to))
        assert lengths.tolist() == [o if t < 0 else t for o, t in zip(old, to)]
        new = [max(0, n - o) for n, o in zip(lengths.tolist(), old)]
        offs = [0]
        for n in new:
            offs.append(offs[-1] + n)
        q, kn, vn = (torch.randn((offs[-1], h * D), generator=g).to(dt) for h in (H, Hk, Hk))
        ca.paged_append_(k, v, kn.cuda(), vn.cuda(), pages, lengths, offsets=ints(offs))
        y = ca.paged_mh_attention(q.cuda(), k, v, pages, lengths, W, H, kv_heads=Hk, sinks=2, offsets=ints(offs), cap=8.0,
                                  slopes=slopes).cpu()
        for b, n in enumerate(lengths.tolist()):
            for kind, x in zip(kept[b], (kn, vn)):
                del kind[n:]
                kind.extend(x[offs[b]:offs[b + 1]])
            if new[b]:
                kb, vb = (torch.stack(x)[None].double() for x in kept[b])
                qb = torch.cat([torch.zeros(n - new[b], H * D), q[offs[b]:offs[b + 1]].float()])[None].double()
                x, bx = M.sliding(qb, kb, vb, W, H, Hk, 2, 1 / math.sqrt(D), None, dt, cap=8.0, slopes=slopes.cpu())[0]
                M.check(y[offs[b]:offs[b + 1]], x[0, n - new[b]:], bx[0, n - new[b]:], f"sequence {b}")
        held = [0] * npages
        for row, n in zip(pages.tolist(), lengths.tolist()):
            for p in row[:P.reach(n, page, most)]:
                held[p] += 1
        same(counts, held)

    step([19, 7, 33])
    for turn in range(6):
        source = [r.randrange(len(kept)) for _ in range(r.choice([4, 6]))]
        pages, lengths, counts = ca.paged_fork(pages, lengths, counts, ints(source), page)
        kept = [[list(x) for x in kept[b]] for b in source]
        step([n + 1 for n in lengths.tolist()])
        step([r.choice([n + 1, n + 5, -1, max(0, n - 3), n + 2]) for n in lengths.tolist()])
        if turn % 2:
            pages, counts = ca.paged_compact_(k, v, pages, counts)
            used = int((counts > 0).sum())
            assert int(pages.max()) < used


def test_captured_calls_follow_their_arrays(ca):
    r = random.Random(9)
    B, most, page, npages, C = 40, 20, 8, 900, 64
    k, v = caches(npages, page, C, torch.bfloat16)
    rows, lengths, counts = pool(r, B, most, page, npages, share=0.5)
    a = [ints(rows), ints(lengths), ints(counts), ints(list(range(B))), ints([-1] * B)]

    def chain():
        forked = ca.paged_fork(*a[:3], a[3], page)
        grown = ca.paged_resize_(k, v, *forked, a[4])
        return (*grown, *ca.paged_compact_(k, v, grown[0], grown[2]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    for _ in range(4):
        rows, lengths, counts = pool(r, B, most, page, npages, share=0.5)
        source = [r.randrange(B) for _ in range(B)]
        to = [r.choice([-1, 0, 30, 100, 160]) for _ in range(B)]
        for t, x in zip(a, (rows, lengths, counts, source, to)):
            t.copy_(torch.tensor(x, dtype=torch.int32))
        fresh = torch.randn((2, *k.shape), generator=torch.Generator().manual_seed(3)).to(k.dtype)
        k.copy_(fresh[0])
        v.copy_(fresh[1])
        graph.replay()
        torch.cuda.synchronize()
        f = P.fork(rows, lengths, counts, source, page)
        *w, moves = P.resize(*f, to, page)
        *z, more = P.compact(w[0], w[2])
        for g, x in zip(out, (*w, *z)):
            same(g, x)
        for t, x in ((k, fresh[0]), (v, fresh[1])):
            assert torch.equal(t.cpu(), moved(moved(x, moves, page), more, page))


def test_a_changed_cache_is_noticed(ca):
    """autograd sees that a saved cache was written."""
    k, v = caches(4, 4, 8, torch.float32)
    w = torch.randn_like(k).requires_grad_(True)
    loss = (w * k).sum()
    ca.paged_compact_(k, v, ints([[3, -1]]), ints([0, 0, 0, 1]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
