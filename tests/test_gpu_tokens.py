"""Token attention, its paged form, the append and rotary positions against the
64-bit restatement of token_model.py, within its element-wise bounds."""
import math

import pytest
import torch

import token_model as M

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def gpu(t, grad=False):
    return t.cuda().requires_grad_(True) if grad else t.cuda()


# B, L, H, Hk, D, W, S, lengths
SHAPES = [
    (1, 1, 1, 1, 8, 1, 0, None),
    (2, 2, 2, 1, 16, 1, 1, None),
    (1, 31, 1, 1, 32, 7, 0, None),
    (1, 32, 4, 2, 64, 32, 5, None),
    (2, 65, 3, 1, 40, 64, 1, None),
    (1, 129, 2, 2, 128, 33, 3, None),
    (1, 200, 7, 1, 64, None, 0, None),
    (3, 150, 6, 2, 80, 20, 17, (150, 71, 1)),
    (3, 97, 4, 4, 96, 96, 2, (0, 97, 96)),
    (1, 333, 4, 1, 104, 65, 70, None),
    (2, 260, 2, 1, 128, 128, 64, (260, 129)),
    (1, 520, 8, 4, 24, 100, 4, None),
    (1, 700, 5, 5, 72, 3, 130, None),
    (1, 1030, 2, 1, 56, 2000, 9, (1025,)),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sliding_values_and_gradients(ca, shape, dtype):
    B, L, H, Hk, D, W, S, lens = shape
    dt = DT[dtype]
    print("sliding", shape, dtype, flush=True)
    q, k, v, dy = (randn(7 + i, B, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H)))
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    tq, tk, tv = (gpu(t, True) for t in (q, k, v))
    kw = dict(kv_heads=Hk, sinks=S, lengths=None if lens is None else lengths.cuda())
    y = ca.sliding_mh_attention(tq, tk, tv, W, H, **kw)
    grads = torch.autograd.grad(y, (tq, tk, tv), dy.cuda())
    with torch.no_grad():
        again = ca.sliding_mh_attention(tq, tk, tv, W, H, **kw)
    assert torch.equal(again, y)
    want = M.sliding(*(t.double() for t in (q, k, v)), W or L, H, Hk, S, 1 / math.sqrt(D), lengths, dt, dy.double())
    for got, (x, bx), name in zip((y, *grads), want, ("y", "dq", "dk", "dv")):
        M.check(got, x, bx, name)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_sliding_padding_may_hold_anything(ca, dtype):
    """Rows behind a signal's length: NaN, infinities and the type's lowest
    value in q, k, v and dy have no influence; outputs there are zero."""
    B, L, H, Hk, D = 3, 100, 4, 2, 64
    dt = DT[dtype]
    lens = torch.tensor([100, 37, 0], dtype=torch.int32)
    base = [randn(3 + i, B, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H))]
    res = []
    for fill in (0.0, math.nan, math.inf, torch.finfo(dt).min):
        t = [x.clone() for x in base]
        for b in range(B):
            for x in t:
                x[b, int(lens[b]):] = fill
        tq, tk, tv = (gpu(x, True) for x in t[:3])
        y = ca.sliding_mh_attention(tq, tk, tv, 16, H, kv_heads=Hk, sinks=3, lengths=lens.cuda())
        res.append([y, *torch.autograd.grad(y, (tq, tk, tv), t[3].cuda())])
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], r))
    for x in res[0]:
        assert torch.isfinite(x).all()
        for b in range(B):
            assert (x[b, int(lens[b]):] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("t", [5, 90, 171])
def test_sliding_other_rows_do_not_feel_a_bad_token(ca, dtype, value, t):
    """A token that is not finite reaches exactly the rows that see it."""
    L, H, Hk, D, W, S = 200, 2, 1, 64, 40, 7
    dt = DT[dtype]
    q, k, v, dy = (randn(11 + i, 1, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H)))
    see = M.visible(torch.arange(L), L, W, S)
    sees_t, seen_by_t = see[:, t], see[t]

    def run(q, k, v, dy):
        tq, tk, tv = (gpu(x, True) for x in (q, k, v))
        y = ca.sliding_mh_attention(tq, tk, tv, W, H, kv_heads=Hk, sinks=S)
        return [x[0].cpu() for x in (y, *torch.autograd.grad(y, (tq, tk, tv), dy.cuda()))]

    # untouched rows: within the bounds of the 64-bit result of the good inputs
    good = [(x[0], bx[0]) for x, bx in M.sliding(*(x.double() for x in (q, k, v)), W, H, Hk, S, 1 / math.sqrt(D), None, dt,
                                                 dy.double())]

    def bad_at(x):
        x = x.clone()
        x[0, t] = value
        return x

    # a key, or a value: rows that see it (y, dq); keys and values that those rows see
    reach = see[sees_t].any(0)
    for args in ((q, bad_at(k), v, dy), (q, k, bad_at(v), dy)):
        got = run(*args)
        for g, r, touched in zip(got, good, (sees_t, sees_t, reach, reach)):
            M.check(g[~touched], r[0][~touched], r[1][~touched], "untouched")
        assert not torch.isfinite(got[0][sees_t]).all(-1).any() or value == math.inf
    # a query, or a row of dy: its own row; the keys and values that it sees
    row = torch.zeros(L, dtype=torch.bool)
    row[t] = True
    for args, y_too in (((bad_at(q), k, v, dy), True), ((q, k, v, bad_at(dy)), False)):
        got = run(*args)
        for g, r, touched in zip(got, good, (row if y_too else row & False, row, seen_by_t, seen_by_t)):
            M.check(g[~touched], r[0][~touched], r[1][~touched], "untouched")


def test_sliding_everything_nan(ca):
    """Inputs that are NaN throughout, as of a run that diverged: NaN results, and
    no row formed again (a second at this size if each were)."""
    q, k, v, dy = (torch.full((1, 2048, 256), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(4))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    e0, e1 = torch.cuda.Event(True), torch.cuda.Event(True)
    for _ in range(2):
        e0.record()
        y = ca.sliding_mh_attention(*leaves, None, 2)
        grads = torch.autograd.grad(y, leaves, dy)
        e1.record()
    torch.cuda.synchronize()
    assert all(torch.isnan(t).all() for t in (y, *grads))
    assert e0.elapsed_time(e1) < 50.0


def test_sliding_float16_gradients_out_of_range(ca):
    """Score gradients that Float16 cannot hold: the rows are formed again in
    Float32; gradients that it cannot hold are infinite."""
    L, H, D, W = 64, 1, 64, 8
    q, k, v = (randn(25 + i, 1, L, D, dtype=torch.float16) for i in range(3))
    dy = randn(28, 1, L, D, dtype=torch.float16) * 3000
    k = k * 0.05
    leaves = [gpu(t, True) for t in (q, k, v)]
    grads = torch.autograd.grad(ca.sliding_mh_attention(*leaves, W, H), leaves, dy.cuda())
    want = M.sliding(*(t.double() for t in (q, k, v)), W, H, H, 0, 1 / math.sqrt(D), None, torch.float16, dy.double())[1:]
    for g, (x, bx), name in zip(grads, want, ("dq", "dk", "dv")):
        inside = x.abs() + bx < 65504
        assert inside.float().mean() > 0.5, name
        g = g.detach().double().cpu()
        assert (torch.isinf(g) | ((g - x).abs() <= bx))[x.abs() + bx >= 65504].all(), name
        M.check(g[inside], x[inside], bx[inside], name)


def test_sliding_rows_past_2_gib(ca):
    """Rows so far apart that a signal spans more than 2^31 bytes."""
    L, H, Hk, D, W, S = 1100, 2, 1, 64, 60, 3
    wide = torch.empty((1, L, 1 << 20), dtype=torch.bfloat16, device="cuda")
    qkv = randn(35, 1, L, (H + 2 * Hk) * D, dtype=torch.bfloat16).cuda()
    far = wide[..., :qkv.shape[-1]]
    far.copy_(qkv)
    dy = wide[..., 4096:4096 + H * D]
    dy.copy_(randn(36, 1, L, H * D, dtype=torch.bfloat16))
    res = []
    for x, g in ((qkv, dy.contiguous()), (far, dy)):
        q, k, v = (t.detach().requires_grad_(True) for t in x.split([H * D, Hk * D, Hk * D], -1))
        y = ca.sliding_mh_attention(q, k, v, W, H, kv_heads=Hk, sinks=S)
        res.append([y, *torch.autograd.grad(y, (q, k, v), g)])
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_sliding_large_scores(ca):
    """Scores of some hundreds, where a row is one key alone, and of the lowest
    values: the running maximum keeps every row finite."""
    L, H, D = 130, 2, 32
    for s in (1e2, 1e-20):
        q, k, v = (randn(21 + i, 1, L, H * D, scale=s if i < 2 else 1.0) for i in range(3))
        y = ca.sliding_mh_attention(*(t.cuda() for t in (q, k, v)), 50, H, sinks=2)
        ((x, bx),) = M.sliding(*(t.double() for t in (q, k, v)), 50, H, H, 2, 1 / math.sqrt(D), None, torch.float32)
        M.check(y, x, bx, f"scale {s}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sliding_strides(ca, dtype):
    """Parts of one projection, transposed and offset views, a batch that is
    expanded: the same result as of copies."""
    B, L, H, Hk, D = 2, 70, 4, 2, 32
    dt = DT[dtype]
    qkv = randn(31, B, L, (H + 2 * Hk) * D, dtype=dt).cuda()
    views = qkv.split([H * D, Hk * D, Hk * D], -1)
    want = ca.sliding_mh_attention(*(t.contiguous() for t in views), 17, H, kv_heads=Hk, sinks=2)
    assert torch.equal(ca.sliding_mh_attention(*views, 17, H, kv_heads=Hk, sinks=2), want)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in views]
    assert torch.equal(ca.sliding_mh_attention(*turned, 17, H, kv_heads=Hk, sinks=2), want)
    strange = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in views]
    assert torch.equal(ca.sliding_mh_attention(*strange, 17, H, kv_heads=Hk, sinks=2), want)
    odd = []
    for t in views:
        buf = torch.zeros(t.numel() + 1, dtype=dt, device="cuda")
        o = buf[1:].view(t.shape)
        o.copy_(t)
        odd.append(o)
    assert torch.equal(ca.sliding_mh_attention(*odd, 17, H, kv_heads=Hk, sinks=2), want)
    # gradients through the split, and of an expanded k, v
    x = qkv.clone().requires_grad_(True)
    y = ca.sliding_mh_attention(*x.split([H * D, Hk * D, Hk * D], -1), 17, H, kv_heads=Hk, sinks=2)
    dy = randn(32, B, L, H * D, dtype=dt).cuda()
    (g,) = torch.autograd.grad(y, x, dy)
    parts = [t.contiguous().requires_grad_(True) for t in views]
    y2 = ca.sliding_mh_attention(*parts, 17, H, kv_heads=Hk, sinks=2)
    assert torch.equal(g, torch.cat(torch.autograd.grad(y2, parts, dy), -1))
    (g2,) = torch.autograd.grad(ca.sliding_mh_attention(*x.split([H * D, Hk * D, Hk * D], -1), 17, H, kv_heads=Hk,
                                                        sinks=2), x, dy.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(g, g2)
    k1 = views[1][:1].contiguous().requires_grad_(True)
    y3 = ca.sliding_mh_attention(views[0], k1.expand(B, -1, -1), views[2], 17, H, kv_heads=Hk)
    k2 = k1.detach().repeat(B, 1, 1).requires_grad_(True)
    y4 = ca.sliding_mh_attention(views[0], k2, views[2], 17, H, kv_heads=Hk)
    assert torch.equal(y3, y4)
    (g3,), (g4,) = torch.autograd.grad(y3, k1, dy), torch.autograd.grad(y4, k2, dy)
    assert torch.equal(g3, g4.sum(0, keepdim=True))


def test_sliding_gradient_against_differences(ca):
    """<grad, direction> against central differences of the kernel's own values:
    within their truncation, taken from a second step width, and the values'
    rounding over the step."""
    L, H, Hk, D, h = 90, 4, 2, 16, 2.0 ** -5
    ts = [randn(41 + i, 1, L, n * D).cuda() for i, n in enumerate((H, Hk, Hk))]
    w = randn(45, 1, L, H * D).cuda()
    leaves = [t.clone().requires_grad_(True) for t in ts]

    def f(args):
        return ca.sliding_mh_attention(*args, 21, H, kv_heads=Hk, sinks=3)

    grads = torch.autograd.grad(f(leaves), leaves, w)
    ((y, by),) = M.sliding(*(t.double().cpu() for t in ts), 21, H, Hk, 3, 1 / math.sqrt(D), None, torch.float32)
    noise = float((w.double().cpu().abs() * by).sum())
    for i in range(3):
        d = randn(50 + i, *ts[i].shape).cuda()

        def slope(step):
            val = [float((f([t + s * step * d if j == i else t for j, t in enumerate(ts)]).double() * w.double()).sum())
                   for s in (1, -1)]
            return (val[0] - val[1]) / (2 * step)

        a, b = slope(h), slope(2 * h)
        got = float((grads[i].double() * d.double()).sum())
        assert abs(got - a) <= abs(a - b) + 2 * noise / h, (i, got, a, b, noise)


def test_sliding_only_some_gradients(ca):
    q, k, v = (randn(61 + i, 2, 40, 64).cuda() for i in range(3))
    dy = randn(64, 2, 40, 64).cuda()
    full = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(ca.sliding_mh_attention(*full, 9, 2), full, dy)
    for i in range(3):
        args = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(ca.sliding_mh_attention(*args, 9, 2), args[i], dy)
        assert torch.equal(g, want[i])
    g = torch.autograd.grad(ca.sliding_mh_attention(*full, 9, 2), full, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), full[0])


@pytest.mark.parametrize("shape", [(0, 5), (2, 0)])
def test_sliding_empty(ca, shape):
    q, k, v = (torch.zeros((*shape, 32), device="cuda", requires_grad=True) for _ in range(3))
    y = ca.sliding_mh_attention(q, k, v, 4, 2)
    assert y.shape == q.shape
    assert all(g.shape == q.shape for g in torch.autograd.grad(y, (q, k, v), torch.zeros_like(y)))


# ---------------------------------------------------------------------------
# paged
# ---------------------------------------------------------------------------
class Case:
    """Sequences of (tokens, new ones) over a cache with pages in random order;
    slots that hold no token are NaN."""

    def __init__(self, seqs, H, Hk, D, page, dt, seed=0, spare=2, pad=0):
        g = torch.Generator().manual_seed(100 + seed)
        need = [-(-n // page) for n, _ in seqs]
        self.pages = torch.full((len(seqs), max(max(need), 1) + 1), -1, dtype=torch.int32)
        order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.pages[b, :n] = order[at:at + n]
            at += n
        C = Hk * D
        self.cache = [torch.full((sum(need) + spare, page, C), math.nan, dtype=dt) for _ in range(2)]
        self.lengths = torch.tensor([n for n, _ in seqs], dtype=torch.int32)
        self.offsets = torch.tensor([0] + [m for _, m in seqs], dtype=torch.int32).cumsum(0).to(torch.int32)
        T = int(self.offsets[-1]) + pad
        self.q = torch.randn(T, H * D, generator=g).to(dt)
        self.new = [torch.randn(T, C, generator=g).to(dt) for _ in range(2)]
        for b, (n, m) in enumerate(seqs):
            for cache, new in zip(self.cache, self.new):
                rows = torch.randn(n, C, generator=g).to(dt)
                if m and n:
                    mm = min(m, n)
                    rows[n - mm:] = new[int(self.offsets[b + 1]) - mm:int(self.offsets[b + 1])]
                for j in range(n):
                    cache[self.pages[b, j // page], j % page] = rows[j]


ONE = [(1, 1), (2, 1), (17, 1), (64, 1), (65, 1), (300, 1)]
# seqs, H, Hk, D, W, S, page, pad
PAGED = [
    ([(1, 1)], 1, 1, 8, 1, 0, 1, 0),
    (ONE, 4, 1, 64, None, 0, 16, 0),
    (ONE, 8, 8, 32, 20, 3, 8, 0),
    (ONE, 40, 1, 40, 64, 4, 64, 0),
    ([(1000, 1), (999, 1), (37, 1)], 16, 2, 128, 256, 4, 32, 0),
    ([(2100, 1)], 5, 1, 96, None, 0, 128, 0),
    ([(0, 1), (5, 1), (0, 1)], 2, 2, 16, 4, 0, 16, 0),
    ([(50, 50)], 4, 2, 64, 13, 2, 16, 0),
    ([(200, 70), (33, 1), (64, 64), (129, 3)], 6, 2, 80, 40, 5, 32, 3),
    ([(200, 1), (400, 129), (10, 0), (7, 7)], 12, 4, 128, None, 0, 16, 1),
    ([(3, 5), (40, 2)], 3, 1, 24, 9, 1, 8, 0),
    ([(1300, 200)], 3, 1, 104, 300, 70, 64, 0),
    ([(90, 9), (600, 9), (1, 1)], 8, 1, 72, 100, 0, 2, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", PAGED, ids=lambda c: str(c)[:60])
def test_paged_values(ca, case, dtype):
    seqs, H, Hk, D, W, S, page, pad = case
    dt = DT[dtype]
    print("paged", case, dtype, flush=True)
    c = Case(seqs, H, Hk, D, page, dt, pad=pad)
    want, bound = M.paged(c.q.double(), *(t.double() for t in c.cache), c.pages, c.lengths, c.offsets, W or 1 << 30, H,
                          Hk, S, 1 / math.sqrt(D), dt)
    args = [t.cuda() for t in (c.q, *c.cache, c.pages, c.lengths)]
    y = ca.paged_mh_attention(*args, W, H, kv_heads=Hk, sinks=S, offsets=c.offsets.cuda())
    M.check(y, want, bound, "y")
    if all(m == 1 for _, m in seqs) and not pad:
        assert torch.equal(ca.paged_mh_attention(*args, W, H, kv_heads=Hk, sinks=S), y)
    # rows behind the last sequence stay as they were in the caller's buffer
    out = torch.full_like(args[0], 7.0)
    assert ca.paged_mh_attention(*args, W, H, kv_heads=Hk, sinks=S, offsets=c.offsets.cuda(), out=out) is out
    T = int(c.offsets[-1])
    assert torch.equal(out[:T], y[:T]) and (out[T:] == 7.0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_then_attend_equals_the_whole_signal(ca, dtype):
    """A signal fed to the cache in chunks and then token by token gives the rows
    of sliding_mh_attention over the whole of it."""
    dt = DT[dtype]
    L, H, Hk, D, W, S, page = 150, 4, 2, 64, 33, 4, 16
    q, k, v = (randn(71 + i, 2, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk)))
    ((want, bound),) = M.sliding(*(t.double() for t in (q, k, v)), W, H, Hk, S, 1 / math.sqrt(D), None, dt)
    M.check(ca.sliding_mh_attention(*(t.cuda() for t in (q, k, v)), W, H, kv_heads=Hk, sinks=S), want, bound, "whole")
    ck, cv = (torch.full((25, page, Hk * D), math.nan, dtype=dt, device="cuda") for _ in range(2))
    pages = torch.randperm(25, generator=torch.Generator().manual_seed(5))[:20].reshape(2, 10).to(torch.int32).cuda()
    done = 0
    for n in (1, 70, 30, 47, 1, 1):
        offs = None if n == 1 else torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
        lens = torch.full((2,), done + n, dtype=torch.int32, device="cuda")
        qq, kk, vv = (t[:, done:done + n].reshape(2 * n, -1).cuda() for t in (q, k, v))
        ca.paged_append_(ck, cv, kk, vv, pages, lens, offsets=offs)
        y = ca.paged_mh_attention(qq, ck, cv, pages, lens, W, H, kv_heads=Hk, sinks=S, offsets=offs)
        M.check(y.reshape(2, n, -1), want[:, done:done + n], bound[:, done:done + n], f"tokens {done}..{done + n}")
        done += n
    assert done == L


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("C", [8, 40, 1, 6])
def test_append_writes_its_slots_alone(ca, dtype, C):
    dt = DT[dtype]
    seqs = [(5, 5), (33, 1), (16, 0), (40, 17), (3, 4)]
    c = Case(seqs, 1, 1, C, 8, dt, pad=2)
    wide = -(-C // 8) * 8  # a cache's rows are 16-byte aligned: a wider row holds the channels
    caches = [torch.full((c.cache[0].shape[0], 8, wide), 3.0, dtype=dt, device="cuda")[..., :C] for _ in range(2)]
    new = [t.cuda() for t in c.new]
    pages = c.pages.clone()
    pages[3, 4] = -1      # the page of tokens 32..39 of the fourth sequence is not there
    pages[1, 4] = 10 ** 6
    ca.paged_append_(*caches, *new, pages.cuda(), c.lengths.cuda(), offsets=c.offsets.cuda())
    want = [torch.full((c.cache[0].shape[0], 8, C), 3.0, dtype=dt) for _ in range(2)]
    for b, (n, m) in enumerate(seqs):
        for i in range(m):
            j = n - m + i
            pg = int(pages[b, j // 8]) if j >= 0 else -1
            if 0 <= pg < want[0].shape[0]:
                for w, t in zip(want, c.new):
                    w[pg, j % 8] = t[int(c.offsets[b]) + i]
    for got, w in zip(caches, want):
        assert torch.equal(got.cpu(), w)


def test_paged_bad_tables_hide_tokens(ca):
    """Page numbers outside the cache, lengths beyond the table, negative and
    zero lengths: nothing outside the cache is read, such tokens are hidden."""
    dt, H, Hk, D, page = torch.bfloat16, 4, 2, 64, 16
    c = Case([(200, 1), (200, 40), (64, 2), (90, 3)], H, Hk, D, page, dt)
    c.pages[0, 3] = -5
    c.pages[1, 11] = 1 << 30
    c.pages[2, :] = -1
    c.pages[3, 0] = c.cache[0].shape[0]
    want, bound = M.paged(c.q.double(), *(t.double() for t in c.cache), c.pages, c.lengths, c.offsets, 1 << 30, H, Hk, 0,
                          1 / math.sqrt(D), dt)
    args = [t.cuda() for t in (c.q, *c.cache, c.pages)]
    y = ca.paged_mh_attention(*args, c.lengths.cuda(), None, H, kv_heads=Hk, offsets=c.offsets.cuda())
    M.check(y, want, bound, "y")
    assert (y[41:43] == 0).all()
    for lens in ([-3, 200, 64, 90], [0, 39, 1, 2], [10 ** 9, 200, 64, 90]):
        y = ca.paged_mh_attention(*args, torch.tensor(lens, dtype=torch.int32, device="cuda"), None, H, kv_heads=Hk,
                                  offsets=c.offsets.cuda())
        assert torch.isfinite(y).all() and (y[0] == 0).all()


@pytest.mark.parametrize("new", [1, 40])
def test_paged_other_rows_do_not_feel_a_bad_token(ca, new):
    """A value that is not finite in a token that some rows see and others do not."""
    dt, H, Hk, D, page, W, S = torch.bfloat16, 4, 2, 64, 16, 30, 2
    c = Case([(200, new), (333, new), (64, min(new, 40))], H, Hk, D, page, dt)
    args = [t.cuda() for t in (c.pages, c.lengths)]
    kw = dict(kv_heads=Hk, sinks=S, offsets=c.offsets.cuda())
    want, bound = M.paged(c.q.double(), *(t.double() for t in c.cache), c.pages, c.lengths, c.offsets, W, H, Hk, S,
                          1 / math.sqrt(D), dt)
    for b, t in ((0, 185), (1, 1), (1, 305), (1, 120), (2, 63)):
        for which in (0, 1):
            cache = [x.clone() for x in c.cache]
            cache[which][c.pages[b, t // page], t % page] = math.nan
            y = ca.paged_mh_attention(c.q.cuda(), *(x.cuda() for x in cache), *args, W, H, **kw)
            seen = torch.zeros(c.q.shape[0], dtype=torch.bool)
            lo, hi, n = int(c.offsets[b]), int(c.offsets[b + 1]), int(c.lengths[b])
            seen[lo:hi] = M.visible(torch.arange(n - (hi - lo), n), n, W, S)[:, t]
            assert torch.isnan(y.cpu()[seen]).all()
            M.check(y[~seen], want[~seen], bound[~seen], f"token {t} of {b}")


def test_paged_many_sequences(ca):
    """More sequences than a wavefront has lanes, some without new tokens."""
    g = torch.Generator().manual_seed(9)
    n = torch.randint(0, 90, (150,), generator=g).tolist()
    seqs = [(t, min(t, int(torch.randint(0, 5, (1,), generator=g)))) for t in n]
    seqs[77] = (260, 100)
    for dtype in (torch.bfloat16, torch.float32):
        c = Case(seqs, 4, 2, 32, 8, dtype, pad=2)
        want, bound = M.paged(c.q.double(), *(t.double() for t in c.cache), c.pages, c.lengths, c.offsets, 25, 4, 2, 3,
                              1 / math.sqrt(32), dtype)
        y = ca.paged_mh_attention(*(t.cuda() for t in (c.q, *c.cache, c.pages, c.lengths)), 25, 4, kv_heads=2, sinks=3,
                                  offsets=c.offsets.cuda())
        M.check(y, want, bound, "y")


def test_paged_views_of_one_cache(ca):
    """k and v as halves of one allocation, by page and by channel."""
    dt, H, Hk, D, page = torch.bfloat16, 4, 2, 32, 16
    c = Case([(100, 1), (70, 12)], H, Hk, D, page, dt)
    args = [t.cuda() for t in (c.pages, c.lengths)]
    kw = dict(kv_heads=Hk, sinks=2, offsets=c.offsets.cuda())
    want = ca.paged_mh_attention(c.q.cuda(), *(t.cuda() for t in c.cache), *args, 30, H, **kw)
    by_page = torch.stack(c.cache, 1).cuda()
    assert torch.equal(ca.paged_mh_attention(c.q.cuda(), by_page[:, 0], by_page[:, 1], *args, 30, H, **kw), want)
    by_channel = torch.cat(c.cache, -1).cuda()
    assert torch.equal(ca.paged_mh_attention(c.q.cuda(), *by_channel.chunk(2, -1), *args, 30, H, **kw), want)
    ca.paged_append_(by_page[:, 0], by_page[:, 1], *(t.cuda() for t in c.new), *args, offsets=c.offsets.cuda())
    assert all(torch.equal(by_page[:, i].cpu().nan_to_num(9.), c.cache[i].nan_to_num(9.)) for i in range(2))


def test_paged_cache_past_4_gib(ca):
    """Rows that lie more than 2^32 bytes into the cache."""
    dt, H, D, page = torch.bfloat16, 2, 128, 64
    npages = (5 << 30) // (page * H * D * 2)
    ck = torch.zeros((npages, page, H * D), dtype=dt, device="cuda")
    cv = torch.zeros_like(ck)
    c = Case([(200, 1), (150, 20)], H, H, D, page, dt)
    far = npages - 1 - c.pages
    far[c.pages < 0] = -1
    for b in range(2):
        for n in range(int(-(-c.lengths[b] // page))):
            ck[int(far[b, n])], cv[int(far[b, n])] = (t[int(c.pages[b, n])].cuda() for t in c.cache)
    kw = dict(sinks=2, offsets=c.offsets.cuda())
    want = ca.paged_mh_attention(c.q.cuda(), *(t.cuda() for t in c.cache), c.pages.cuda(), c.lengths.cuda(), 70, H, **kw)
    assert torch.equal(ca.paged_mh_attention(c.q.cuda(), ck, cv, far.cuda(), c.lengths.cuda(), 70, H, **kw), want)
    ck.zero_(), cv.zero_()
    ca.paged_append_(ck, cv, *(t.cuda() for t in c.new), far.cuda(), c.lengths.cuda(), offsets=c.offsets.cuda())
    assert torch.equal(ck[int(far[0, 3]), 199 % page].cpu(), c.new[0][0])


# ---------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------
# (B, *spatial slow first), H, D, pairs
ROTARY = [
    ((1, 1), 1, 2, (1,)),
    ((2, 33), 3, 16, (8,)),
    ((2, 9, 7), 4, 16, (4, 4)),
    ((1, 30, 41), 2, 64, (16, 12)),
    ((2, 3, 5, 4), 2, 128, (22, 21, 16)),
    ((1, 2, 17, 9), 5, 40, (8, 4, 8)),
    ((3, 300), 1, 104, (17,)),
    ((1, 4, 4), 7, 256, (64, 64)),
]


def grid_positions(spatial):
    axes = [torch.arange(n) for n in spatial]
    return torch.stack(list(reversed(torch.meshgrid(*axes, indexing="ij"))), -1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", ROTARY, ids=str)
def test_rotary_values_and_gradients(ca, case, dtype, interleaved):
    shape, H, D, pairs = case
    dt = DT[dtype]
    x, dy = randn(81, *shape, H * D, dtype=dt), randn(82, *shape, H * D, dtype=dt)
    own = grid_positions(shape[1:])
    shared = torch.randint(-50000, 50000, own.shape, generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    each = torch.randint(0, 1000, (*shape, len(pairs)), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    for given, pos in ((None, own), (shared, shared), (each, each)):
        t = gpu(x, True)
        y = ca.axial_rotary(t, pairs, H, positions=None if given is None else given.cuda(), interleaved=interleaved)
        (g,) = torch.autograd.grad(y, t, dy.cuda())
        M.check(y, *M.rotary(x.double(), pairs, H, 10000.0, pos, interleaved, dt), "y")
        M.check(g, *M.rotary(dy.double(), pairs, H, 10000.0, pos, interleaved, dt, inverse=True), "dx")


def test_rotary_far_positions(ca):
    pos = torch.tensor([[0], [1], [-1], [2 ** 24 + 1], [2 ** 31 - 1], [-2 ** 31], [1 << 30]], dtype=torch.int32)
    x = randn(83, 7, 2 * 32)
    y = ca.axial_rotary(x.cuda(), (16,), 2, positions=pos.cuda(), base=500000.0)
    M.check(y, *M.rotary(x.double(), (16,), 2, 500000.0, pos, False, torch.float32), "y")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rotary_strides(ca, dtype):
    dt = DT[dtype]
    qkv = randn(84, 2, 6, 5, 3 * 64, dtype=dt).cuda()
    want = [ca.axial_rotary(t.contiguous(), (8, 8), 2) for t in qkv.chunk(3, -1)]
    for t, w in zip(qkv.chunk(3, -1), want):
        assert torch.equal(ca.axial_rotary(t, (8, 8), 2), w)
        assert torch.equal(ca.axial_rotary(t.transpose(1, 2).contiguous().transpose(1, 2), (8, 8), 2), w)
    odd = torch.zeros(want[0].numel() + 1, dtype=dt, device="cuda")[1:].view(want[0].shape)
    odd.copy_(qkv[..., :64])
    assert torch.equal(ca.axial_rotary(odd, (8, 8), 2), want[0])
    one = qkv[:1, :1, :1, :64]
    assert torch.equal(ca.axial_rotary(one, (8, 8), 2), want[0][:1, :1, :1])
    assert ca.axial_rotary(qkv[:, :0, :, :64], (8, 8), 2).shape == (2, 0, 5, 64)


# ---------------------------------------------------------------------------
# streams, graphs, the run of them
# ---------------------------------------------------------------------------
def test_on_another_stream(ca):
    q, k, v = (randn(91 + i, 1, 300, 128, dtype=torch.bfloat16).cuda() for i in range(3))
    want = ca.sliding_mh_attention(q, k, v, 64, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = [t.clone() for t in (q, k, v)]
        got = ca.sliding_mh_attention(*x, 64, 2)
        r = ca.axial_rotary(x[0], (16,), 2)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(r, ca.axial_rotary(q, (16,), 2))


def test_training_step_graph_replays(ca):
    """Rotary on q and k, the attention and all gradients captured; replays on
    new inputs, with eager work between, equal the eager results."""
    B, L, H, Hk, D = 2, 200, 4, 2, 64
    lens = torch.tensor([200, 130], dtype=torch.int32, device="cuda")

    def step(x, dy):
        x = x.detach().requires_grad_(True)
        q, k, v = x.split([H * D, Hk * D, Hk * D], -1)
        q, k = ca.axial_rotary(q, (32,), H), ca.axial_rotary(k, (32,), Hk)
        y = ca.sliding_mh_attention(q, k, v, 50, H, kv_heads=Hk, sinks=4, lengths=lens)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    def inputs(i):
        return (randn(95 + i, B, L, (H + 2 * Hk) * D, dtype=torch.bfloat16).cuda(),
                randn(195 + i, B, L, H * D, dtype=torch.bfloat16).cuda())

    x, dy = inputs(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x, dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(x, dy)
    for i in range(4):
        nx, ndy = inputs(i)
        lens.copy_(torch.tensor([200 - i, 130 + i], dtype=torch.int32))
        want = step(nx, ndy)
        x.copy_(nx), dy.copy_(ndy)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_two_decoding_graphs_share_a_pool(ca):
    """Append and attention of single tokens captured twice into one memory pool
    (the second graph's workspace may lie where the first one's did); replays in
    turn follow the lengths and pages that the arrays hold then."""
    dt, H, Hk, D, page, B = torch.bfloat16, 8, 2, 128, 16, 3
    ck, cv = (torch.zeros((120, page, Hk * D), dtype=dt, device="cuda") for _ in range(2))
    pages = torch.randperm(120, generator=torch.Generator().manual_seed(3))[:90].reshape(B, 30).to(torch.int32).cuda()
    fill = [randn(200 + i, 120, page, Hk * D, dtype=dt).cuda() for i in range(2)]
    ck.copy_(fill[0]), cv.copy_(fill[1])
    lens = torch.tensor([400, 17, 250], dtype=torch.int32, device="cuda")
    q, k, v = (randn(205 + i, B, h * D, dtype=dt).cuda() for i, h in enumerate((H, Hk, Hk)))

    def step(W):
        ca.paged_append_(ck, cv, k, v, pages, lens)
        return ca.paged_mh_attention(q, ck, cv, pages, lens, W, H, kv_heads=Hk, sinks=4)

    step(None), step(100)
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for W in (None, 100):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(step(W))
        graphs.append(g)
    for i in range(4):
        lens.add_(1)
        for t, seed in ((q, 300), (k, 310), (v, 320)):
            t.copy_(randn(seed + i, *t.shape, dtype=dt))
        for W, g, out in zip((None, 100), graphs, outs):
            want = step(W)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), (i, W)


def plain_block(m, x, lens=None):
    """SlidingAttBlock in 64 bits on the CPU."""
    x = x.double().cpu()
    q, k, v = (x @ m.qkv.weight.double().cpu().T + m.qkv.bias.double().cpu()).split(m.parts, -1)
    pos = torch.arange(x.shape[1])[:, None]
    q, k = (M.rotary(t, m.rotary, h, m.base, pos, False, torch.float32)[0] for t, h in ((q, m.nheads), (k, m.kv_heads)))
    D = q.shape[-1] // m.nheads
    ((y, _),) = M.sliding(q, k, v, m.window, m.nheads, m.kv_heads, m.sinks, 1 / math.sqrt(D), lens, torch.float32)
    return x + y @ m.o.weight.double().cpu().T + m.o.bias.double().cpu()


def test_block_trains_and_serves(ca):
    """The layer's forward, its gradients (against a plain composition's
    differences of a Float64 copy) and its step, token by token and in chunks."""
    torch.manual_seed(0)
    C, L, page = 64, 60, 8
    m = ca.SlidingAttBlock(C, 16, nheads=4, kv_heads=2, sinks=2, rotary=(8,)).cuda()
    x = randn(400, 2, L, C).cuda()
    xg = x.clone().requires_grad_(True)
    y = m(xg)
    want = plain_block(m, x)
    # Float32 projections of 64 channels around the attention: 3 * 64 products' roundings
    want = want.detach()
    tol = 400 * 2.0 ** -24 * float(want.abs().max() + 4)
    assert float((y.detach().double().cpu() - want).abs().max()) <= tol
    w = randn(401, 2, L, C).cuda()
    (g,) = torch.autograd.grad(y, xg, w)
    d, h = randn(402, 2, L, C).cuda(), 2.0 ** -8
    slope = [float(((plain_block(m, x + s * h * d) - plain_block(m, x - s * h * d)) * w.double().cpu()).sum()) / (2 * s * h)
             for s in (1, 2)]
    got = float((g.double() * d.double()).sum())
    size = float((w.abs().sum() * 4))
    assert abs(got - slope[0]) <= abs(slope[0] - slope[1]) + 400 * 2.0 ** -24 * size
    ck, cv = (torch.full((20, page, 32), math.nan, device="cuda") for _ in range(2))
    pages = torch.arange(16, dtype=torch.int32).flip(0).reshape(2, 8).contiguous().cuda()
    n = 40
    offs = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    pos = torch.arange(n, dtype=torch.int32).repeat(2)[:, None].cuda()
    out = m.step(x[:, :n].reshape(2 * n, C), ck, cv, pages, torch.full((2,), n, dtype=torch.int32, device="cuda"), offs, pos)
    assert float((out.reshape(2, n, C).double().cpu() - want[:, :n]).abs().max()) <= tol
    for i in range(n, L):
        out = m.step(x[:, i], ck, cv, pages, torch.full((2,), i + 1, dtype=torch.int32, device="cuda"))
        assert float((out.double().cpu() - want[:, i]).abs().max()) <= tol, i
    with pytest.raises(AssertionError, match="positions"):
        m.step(x[:, 0], ck, cv, pages, pages[:, 0], offs)


def test_image_block_with_rotary(ca):
    """CircAttBlock(rotary=...): the fused attention on turned queries and keys."""
    torch.manual_seed(1)
    m = ca.CircAttBlock(32, 7, 2, rotary=(4, 4)).cuda()
    x = randn(410, 2, 12, 14, 32).cuda().requires_grad_(True)
    y = m(x)
    q, k = (ca.axial_rotary(f(x), (4, 4), 2) for f in (m.q, m.k))
    z, _ = ca.circulant_mh_attention(ca.DotSimilarity(), q, k, m.v(x), 7, 2, materialize=False, channels_last=True)
    want = x + m.o(z)
    assert torch.equal(y, want)
    dy = randn(411, *y.shape).cuda()
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(want, x, dy)[0])
    plain = ca.CircAttBlock(32, 7, 2).cuda()
    plain.load_state_dict(m.state_dict())
    assert not torch.equal(plain(x), y)


def test_refusals_on_device_tensors(ca):
    x = torch.zeros(2, 8, 64, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    cases = [
        (AssertionError, "divisible", lambda: ca.sliding_mh_attention(x, x, x, 3, 5)),
        (AssertionError, "kv_heads", lambda: ca.sliding_mh_attention(x, x, x, 3, 4, kv_heads=3)),
        (AssertionError, "k and v must be", lambda: ca.sliding_mh_attention(x, x, x, 3, 4, kv_heads=2)),
        (AssertionError, "type", lambda: ca.sliding_mh_attention(x, x.half(), x, 3, 2)),
        (TypeError, "float32", lambda: ca.sliding_mh_attention(x.double(), x, x, 3, 2)),
        (AssertionError, "window", lambda: ca.sliding_mh_attention(x, x, x, 0, 2)),
        (AssertionError, "sinks", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, sinks=-1)),
        (AssertionError, "scale", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, scale=-1.0)),
        (TypeError, "int32", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, lengths=torch.zeros(2, device="cuda"))),
        (AssertionError, "shape", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, lengths=torch.zeros(3, **i32))),
        (AssertionError, "device", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, lengths=torch.zeros(2, dtype=torch.int32))),
        (NotImplementedError, "multiple of 8", lambda: ca.sliding_mh_attention(x, x, x, 3, 16)),
        (AssertionError, "token signals", lambda: ca.sliding_mh_attention(x[0], x[0], x[0], 3, 2)),
        (AssertionError, "axes", lambda: ca.axial_rotary(x, (4, 4), 2)),
        (AssertionError, "do not fit", lambda: ca.axial_rotary(x, (17,), 2)),
        (AssertionError, "shape", lambda: ca.axial_rotary(x, (4,), 2, positions=torch.zeros(8, 2, **i32))),
        (TypeError, "int32", lambda: ca.axial_rotary(x, (4,), 2, positions=torch.zeros(8, 1, device="cuda"))),
    ]
    q, cache, pages, lens = x[:, 0], torch.zeros(4, 16, 64, device="cuda"), torch.zeros(2, 2, **i32), torch.ones(2, **i32)

    def paged(q=q, ck=cache, cv=cache, pages=pages, lens=lens, **kw):
        return ca.paged_mh_attention(q, ck, cv, pages, lens, 8, 2, **kw)

    cases += [
        (AssertionError, "the caches must hold", lambda: paged(ck=cache[..., :32], cv=cache[..., :32])),
        (AssertionError, "alike", lambda: paged(cv=cache[:2])),
        (NotImplementedError, "power of two", lambda: paged(ck=cache[:, :12], cv=cache[:, :12])),
        (TypeError, "pages", lambda: paged(pages=pages.long())),
        (AssertionError, "lengths", lambda: paged(lens=lens[:1])),
        (AssertionError, "offsets", lambda: paged(offsets=lens)),
        (AssertionError, "without offsets", lambda: paged(q=x[0])),
        (AssertionError, "out", lambda: paged(out=torch.zeros(3, 64, device="cuda"))),
        (AssertionError, "k and v must be", lambda: ca.paged_append_(cache, cache.clone(), q[:, :32], q[:, :32], pages, lens)),
    ]
    for kind, text, call in cases:
        with pytest.raises(kind, match=text):
            call()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("W,sharp", [(2, 1.0), (512, 4.0), (512, 8.0)])
def test_query_gradient_of_few_effective_keys(ca, dtype, W, sharp):
    """dq where few keys carry a row (a short window, or a softmax with sharp
    peaks) and the score gradients cancel most.  Three roundings of at most u =
    eps/2 enter, of dS, of P by way of y, and of the result, with mean squares of
    at most u^2/3 each (uniform in a step): together ||error|| <= u ||dq||.  A d =
    <dy, y> of the rounded y exceeds it: 1.3 u at the sharpest."""
    B, n, D = 1, 512, 64
    q, k, v, g = (randn(731 + i, B, n, D, dtype=dtype) * (sharp if i == 0 else 1) for i in range(4))
    x = [t.cuda().requires_grad_() for t in (q, k, v)]
    y = ca.sliding_mh_attention(*x, W, 1)
    (dq,) = torch.autograd.grad(y, x[:1], g.cuda())
    q, k, v, g = (t[0].double() for t in (q, k, v, g))
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    p = (q @ k.T * D ** -0.5).masked_fill((j > i) | (j <= i - W), -math.inf).softmax(-1)
    dp = g @ v.T
    want = p * (dp - (p * dp).sum(-1, keepdim=True)) @ k * D ** -0.5
    u = torch.finfo(dtype).eps / 2
    assert (dq[0].cpu().double() - want).norm() <= u * want.norm(), (dq[0].cpu().double() - want).norm() / want.norm() / u
