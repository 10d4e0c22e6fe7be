"""Sequences that drop tokens and bring new ones in one step: resized to what stays, then to
that with the new ones, no page is written that another sequence holds."""
import random

import pytest
import torch

import pages_model as P


def written(rows, before, after, page):
    """(page, slot) of every token that an append writes, by sequence."""
    return [[(row[t // page], t % page) for t in range(a, n)] for row, a, n in zip(rows, before, after)]


def test_two_resizes_over_lists():
    """Over lists, for many pools: the slots of the new tokens are nobody else's, and what stays is
    where it was or a copy of it."""
    r = random.Random(2)
    page, most = 8, 10
    for _ in range(200):
        n, B = r.randint(1, 60), r.randint(2, 5)
        npages = -(-n // page) + 30
        order = list(range(npages))
        r.shuffle(order)
        row = order[:-(-n // page)]
        rows, lengths = [row + [-1] * (most - len(row))], [n]
        counts = [int(p in row) for p in range(npages)]
        rows, lengths, counts = P.fork(rows, lengths, counts, [0] * B, page)
        stays = [r.randint(0, n) for _ in range(B)]
        rows, lengths, counts, moves = P.resize(rows, lengths, counts, stays, page)
        assert not moves and lengths == stays
        rows, lengths, counts, moves = P.resize(rows, lengths, counts, [s + r.randint(1, 9) for s in stays], page)
        for b, slots in enumerate(written(rows, stays, lengths, page)):
            for c in range(B):
                if c != b:
                    theirs = {(rows[c][t // page], t % page) for t in range(lengths[c])}
                    assert not theirs & set(slots)


def test_one_resize_shrinks():
    """One resize to fewer tokens leaves the shared page shared: a new token among them has
    another sequence's slot."""
    rows, lengths, counts = P.fork([[0, 1, 2]], [20], [1, 1, 1, 0], [0, 0], 8)
    rows, lengths, counts, moves = P.resize(rows, lengths, counts, [-1, 18], 8)
    assert not moves and rows[0] == rows[1] == [0, 1, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("stays,new", [(17, 1), (16, 3), (3, 1), (0, 2), (20, 1), (19, 9)])
def test_a_rollback_with_new_tokens(cuda, stays, new):
    """The sibling's tokens stay, and both are attended right."""
    import circulant_attention as ca
    import shaped_model as M
    H, D, page, n, dt = 2, 32, 8, 20, torch.bfloat16
    g = torch.Generator().manual_seed(stays)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    old, fresh = (torch.randn((2, m, H * D), generator=g).to(dt) for m in (n, new))
    k, v = (torch.zeros((12, page, H * D), dtype=dt, device="cuda") for _ in range(2))
    pages, lengths, counts = ca.paged_resize_(k, v, ints([[-1] * 5]), ints([0]), ints([0] * 12), ints([n]))
    ca.paged_append_(k, v, *old.cuda(), pages, lengths, offsets=ints([0, n]))
    pages, lengths, counts = ca.paged_fork(pages, lengths, counts, ints([0, 0]), page)
    pages, lengths, counts = ca.paged_resize_(k, v, pages, lengths, counts, ints([-1, stays]))
    pages, lengths, counts = ca.paged_resize_(k, v, pages, lengths, counts, ints([-1, stays + new]))
    assert lengths.tolist() == [n, stays + new]
    ca.paged_append_(k, v, *fresh.cuda(), pages, lengths, offsets=ints([0, 0, new]))
    tokens = [old, torch.cat([old[:, :stays], fresh], 1)]
    for b, t in enumerate(tokens):
        for cache, want in zip((k, v), t):
            got = torch.stack([cache[pages[b, i // page], i % page] for i in range(t.shape[1])]).cpu()
            assert torch.equal(got, want), f"sequence {b}"
    q = torch.randn((2, H * D), generator=g).to(dt)
    y = ca.paged_mh_attention(q.cuda(), k, v, pages, lengths, 64, H).cpu()
    x, bx = M.paged(q.double(), k.cpu().double(), v.cpu().double(), pages.cpu(), lengths.cpu(), torch.arange(3), 64, H, H, 0,
                    D ** -0.5, dt)
    M.check(y, x, bx, "attention")
