"""sliding_mh_attention and paged_mh_attention with shaped scores (cap, slopes,
documents, prefix) against the 64-bit restatement of shaped_model.py, within its
element-wise bounds."""
import math
import random

import pytest
import torch

import shaped_model as M

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def geometric(H):
    return torch.exp2(-8.0 * torch.arange(1, H + 1, dtype=torch.float64) / H).float()


def places_of(docs, L):
    """(B, L) places of documents of the given lengths, the last one cut or drawn out."""
    rows = []
    for d in docs:
        row = [i for n in d for i in range(n)][:L]
        rows.append(row + list(range(L - len(row))))
    return torch.tensor(rows, dtype=torch.int32)


def run(ca, q, k, v, dy, W, H, Hk, S, lengths, shape, grad=True):
    dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in shape.items()}
    leaves = [t.cuda().requires_grad_(grad) for t in (q, k, v)]
    y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=Hk, sinks=S, lengths=None if lengths is None else lengths.cuda(), **dev)
    return (y, *torch.autograd.grad(y, leaves, dy.cuda())) if grad else (y,)


def compare(ca, B, L, H, Hk, D, W, S, lens, dt, shape, loud=1.0, seed=7):
    q, k, v, dy = (randn(seed + i, B, L, h * D, dtype=dt, scale=loud if i == 0 else 1.0)
                   for i, h in enumerate((H, Hk, Hk, H)))
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    got = run(ca, q, k, v, dy, W, H, Hk, S, lengths, shape)
    (again,) = run(ca, q, k, v, dy, W, H, Hk, S, lengths, shape, grad=False)
    assert torch.equal(again, got[0])
    want = M.sliding(*(t.double() for t in (q, k, v)), W or L, H, Hk, S, 1 / math.sqrt(D), lengths, dt, dy=dy.double(), **shape)
    for g, (x, bx), name in zip(got, want, ("y", "dq", "dk", "dv")):
        M.check(g, x, bx, name)


# B, L, H, Hk, D, W, S, lengths
SHAPES = [
    (1, 1, 1, 1, 8, 1, 0, None),
    (2, 2, 2, 1, 16, 1, 1, None),
    (1, 31, 1, 1, 32, 7, 0, None),
    (1, 65, 4, 2, 64, 32, 5, None),
    (1, 129, 2, 2, 128, 33, 3, None),
    (1, 200, 7, 1, 64, None, 0, None),
    (3, 150, 6, 2, 80, 20, 17, (150, 71, 1)),
    (3, 97, 4, 4, 96, 96, 2, (0, 97, 96)),
    (1, 333, 4, 1, 104, 65, 70, None),
    (2, 260, 2, 1, 128, 128, 64, (260, 129)),
    (1, 700, 5, 5, 72, 3, 130, None),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap,biased", [(15.0, False), (15.0, True), (300.0, False), (300.0, True), (0.0, True)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_caps_and_slopes(ca, shape, biased, cap, dtype):
    B, L, H, Hk, D, W, S, lens = shape
    print("shaped", shape, cap, biased, dtype, flush=True)
    compare(ca, B, L, H, Hk, D, W, S, lens, DT[dtype], {"cap": cap or None, "slopes": geometric(H) if biased else None},
            loud=4.0 if cap == 15.0 else 1.0)


DOCS = [
    # B, L, H, Hk, D, W, S, lengths, documents
    (1, 40, 2, 1, 32, None, 0, None, [[1] * 40]),
    (1, 65, 4, 2, 64, 32, 5, None, [[3, 1, 30, 20]]),
    (2, 200, 3, 1, 40, 9, 2, None, [[64, 64, 64], [5, 190]]),
    (1, 333, 4, 1, 104, None, 0, None, [[100, 33, 128, 1, 2, 60]]),
    (2, 300, 8, 2, 128, 50, 70, (300, 111), [[129, 1, 100], [10, 80, 100]]),
    (1, 700, 5, 5, 72, 3, 130, None, [[7, 300, 128, 200]]),
    (1, 1030, 2, 1, 56, 200, 4, None, [[31, 33, 400, 64, 500]]),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 15.0])
@pytest.mark.parametrize("shape", DOCS, ids=str)
def test_documents(ca, shape, cap, dtype):
    B, L, H, Hk, D, W, S, lens, docs = shape
    print("documents", shape, cap, dtype, flush=True)
    compare(ca, B, L, H, Hk, D, W, S, lens, DT[dtype],
            {"cap": cap or None, "slopes": geometric(H) if cap else None, "places": places_of(docs, L)})


PREFIXES = [
    # B, L, H, Hk, D, W, S, lengths, prefix
    (1, 1, 1, 1, 8, 1, 0, None, [1]),
    (1, 40, 2, 1, 32, None, 0, None, [40]),
    (2, 65, 4, 2, 64, 32, 5, None, [3, 0]),
    (3, 150, 6, 2, 80, 20, 17, (150, 71, 1), [64, 200, -5]),
    (1, 333, 4, 1, 104, 65, 70, None, [130]),
    (2, 400, 2, 1, 128, 30, 0, (400, 129), [257, 128]),
    (1, 700, 5, 5, 72, 3, 130, None, [300]),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 15.0])
@pytest.mark.parametrize("shape", PREFIXES, ids=str)
def test_prefixes(ca, shape, cap, dtype):
    B, L, H, Hk, D, W, S, lens, prefix = shape
    print("prefix", shape, cap, dtype, flush=True)
    compare(ca, B, L, H, Hk, D, W, S, lens, DT[dtype],
            {"cap": cap or None, "slopes": geometric(H) if cap else None, "prefix": torch.tensor(prefix, dtype=torch.int32)})


@pytest.mark.parametrize("seed", range(30))
def test_drawn(ca, seed):
    r = random.Random(seed)
    dt = DT[r.choice(["f32", "f16", "bf16"])]
    D, Hk, G = r.choice([8, 16, 24, 32, 40, 64, 72, 96, 104, 128]), r.choice([1, 2, 3]), r.choice([1, 2, 3, 5, 8])
    B, L = r.choice([1, 2, 3]), int(2 ** r.uniform(0, 9.5))
    W, S = r.choice([None, int(2 ** r.uniform(0, 9))]), r.choice([0, 0, 3, r.randint(1, 200)])
    lens = [L] + [r.randint(0, L) for _ in range(B - 1)] if r.random() < 0.4 else None
    shape = {"cap": r.choice([None, 5.0, 30.0, 1000.0])}
    if r.random() < 0.5:
        shape["slopes"] = geometric(G * Hk)
    kind = r.choice(["", "places", "prefix"])
    if kind == "places":
        shape["places"] = places_of([[r.randint(1, 2 * max(1, L // 4)) for _ in range(40)] for _ in range(B)], L)
    if kind == "prefix":
        shape["prefix"] = torch.tensor([r.randint(0, L) for _ in range(B)], dtype=torch.int32)
    if len(shape) == 1 and shape["cap"] is None:
        shape["cap"] = 20.0
    print("drawn", seed, B, L, Hk * G, Hk, D, W, S, lens, kind, shape["cap"], dt, flush=True)
    compare(ca, B, L, Hk * G, Hk, D, W, S, lens, dt, shape, loud=3.0, seed=seed)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_against_differences(ca, dtype):
    """Central differences of the 64-bit form and of the kernels' own gradients."""
    B, L, H, Hk, D = 1, 50, 4, 2, 32
    dt = DT[dtype]
    q, k, v, dy = (randn(31 + i, B, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H)))
    shape = {"cap": 3.0, "slopes": geometric(H), "places": places_of([[20, 7, 23]], L)}
    grads = run(ca, q, k, v, dy, 12, H, Hk, 2, None, shape)[1:]
    # the bounds of every element of the gradient, along the direction
    want = M.sliding(*(t.double() for t in (q, k, v)), 12, H, Hk, 2, 1 / math.sqrt(D), None, dt, dy=dy.double(), **shape)[1:]
    for at, (g, (_, bg)) in enumerate(zip(grads, want)):
        h = randn(50 + at, *g.shape).double()
        step, vals = 1e-4, []
        for sign in (1, -1):
            args = [t.double() for t in (q, k, v)]
            args[at] = args[at] + sign * step * h
            vals.append((M.sliding(*args, 12, H, Hk, 2, 1 / math.sqrt(D), None, dt, **shape)[0][0] * dy.double()).sum())
        slope = float(vals[0] - vals[1]) / (2 * step)
        # differences in 64 bits: step^2 times the third derivative, below 1e-6 here
        assert abs(float((g.double().cpu() * h).sum()) - slope) <= float((bg * h.abs()).sum()) + 1e-5 * (1 + abs(slope))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf, "lowest"])
def test_other_documents_may_hold_anything(ca, dtype, fill):
    """What one document holds reaches no other: bounds as if it held zeros."""
    L, H, Hk, D = 230, 4, 2, 64
    dt = DT[dtype]
    fill = torch.finfo(dt).min if fill == "lowest" else fill
    docs = [40, 65, 3, 122]
    places = places_of([docs], L)
    base = [randn(3 + i, 1, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H))]
    at = 0
    for n in docs:
        for W, S in ((None, 0), (16, 3)):
            for cap in (None, 15.0):
                t = [x.clone() for x in base]
                for x in t:
                    x[0, at:at + n] = fill
                shape = {"cap": cap, "slopes": geometric(H) if cap else None, "places": places}
                got = run(ca, *t, W, H, Hk, S, None, shape)
                clean = [x.clone() for x in base]
                for x in clean:
                    x[0, at:at + n] = 0
                want = M.sliding(*(x.double() for x in clean[:3]), W or L, H, Hk, S, 1 / math.sqrt(D), None, dt,
                                 dy=clean[3].double(), **shape)
                keep = torch.ones(L, dtype=torch.bool)
                keep[at:at + n] = False
                for g, (x, bx), name in zip(got, want, ("y", "dq", "dk", "dv")):
                    M.check(g[:, keep], x[:, keep], bx[:, keep], name)
        at += n


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("t", [5, 90, 171])
@pytest.mark.parametrize("kind", ["bias", "prefix", "places"])
def test_a_bad_token_reaches_those_that_see_it(ca, dtype, value, t, kind):
    L, H, Hk, D, W, S = 200, 2, 1, 64, 40, 7
    dt = DT[dtype]
    shape = {"cap": 10.0, "slopes": geometric(H)}
    start, P = None, 0
    if kind == "prefix":
        P = 80
        shape["prefix"] = torch.tensor([P], dtype=torch.int32)
    if kind == "places":
        shape["places"] = places_of([[60, 30, 110]], L)
        start = torch.arange(L) - shape["places"][0]
    q, k, v, dy = (randn(11 + i, 1, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H)))
    see = M.visible(torch.arange(L), L, W, S, start, P)
    sees_t, seen_by_t = see[:, t], see[t]
    good = M.sliding(*(x.double() for x in (q, k, v)), W, H, Hk, S, 1 / math.sqrt(D), None, dt, dy=dy.double(), **shape)

    def bad_at(x):
        x = x.clone()
        x[0, t] = value
        return x

    reach = see[sees_t].any(0)
    row = torch.zeros(L, dtype=torch.bool)
    row[t] = True
    for args, touched in (((q, bad_at(k), v, dy), (sees_t, sees_t, reach, reach)),
                          ((q, k, bad_at(v), dy), (sees_t, sees_t, reach, reach)),
                          ((bad_at(q), k, v, dy), (row, row, seen_by_t, seen_by_t)),
                          ((q, k, v, bad_at(dy)), (row & False, row, seen_by_t, seen_by_t))):
        got = run(ca, *args, W, H, Hk, S, None, shape)
        for g, (x, bx), hit in zip(got, good, touched):
            M.check(g[:, ~hit], x[:, ~hit], bx[:, ~hit], "untouched")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_beyond_the_type_are_the_cap(ca, dtype, sign):
    """Products that overflow: all scores are the cap (or its negative), and the row the
    mean of the values that it sees."""
    L, D = 70, 32
    dt = DT[dtype]
    q = torch.zeros(1, L, D, dtype=dt)
    k = torch.zeros(1, L, D, dtype=dt)
    q[..., 0], k[..., 0] = 1e30, sign * 1e30
    v, dy = randn(1, 1, L, D, dtype=dt), randn(2, 1, L, D, dtype=dt)
    compare_at = M.sliding(*(t.double() for t in (q, k, v)), L, 1, 1, 0, 1 / math.sqrt(D), None, dt, cap=7.0)
    y, dq, dk, dv = run(ca, q, k, v, dy, None, 1, 1, 0, None, {"cap": 7.0})
    # (the bound of the model counts the products' rounding, which does not matter here)
    mean = torch.cumsum(v.double(), 1) / torch.arange(1, L + 1)[None, :, None]
    assert (compare_at[0][0] - mean).abs().max() < 1e-12
    size = torch.cumsum(v.double().abs(), 1) / torch.arange(1, L + 1)[None, :, None]
    M.check(y, mean, (2 * M.HALF[dt] + (L + 16) * M.F) * size + 1e-6, "y")
    assert (dq == 0).all() and (dk == 0).all() and torch.isfinite(dv).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap,loud", [(20.0, 0.5), (20.0, 3.0), (20.0, 30.0), (400.0, 2.0), (400.0, 60.0), (400.0, 600.0),
                                      (1e4, 1.0), (1e6, 1.0), (0.05, 1.0), (1e-4, 1.0)])
def test_all_reaches_of_the_curve(ca, cap, loud, dtype):
    """Scores far below the cap, about it and beyond it; caps that leave nothing and that
    leave everything as it is."""
    compare(ca, 1, 150, 2, 1, 64, 70, 3, None, DT[dtype], {"cap": cap}, loud=loud)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e30, 1e-25])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("biased", [False, True])
def test_capped_values_of_any_size(ca, biased, sign, size, dtype):
    """Values near the ends of Float32 under scores near the cap's: the weights' reference
    must not cost their range.  Prompt, single tokens and chunks; half of the keys at one
    end of the cap, half at the other, the first tiles at the lower one."""
    L, H, D, page, dt = 400, 2, 64, 16, DT[dtype]
    q, k = (randn(5 + i, 1, L, H * D, dtype=dt, scale=0.1) for i in range(2))
    q.view(1, L, H, D)[..., 0] = 40.0
    k.view(1, L, H, D)[..., 0] = 40.0 * sign * torch.where(torch.arange(L) < L // 2, -1.0, 1.0)[None, :, None]
    v = randn(9, 1, L, H * D, dtype=dt, scale=size)
    sh = {"cap": 60.0, "slopes": torch.tensor([0.01, 0.002]) if biased else None}
    want = M.sliding(*(t.double() for t in (q, k, v)), L, H, H, 0, 1 / math.sqrt(D), None, dt, **sh)[0]
    dev = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in sh.items()}
    with torch.no_grad():
        y = ca.sliding_mh_attention(q.cuda(), k.cuda(), v.cuda(), None, H, **dev)
    M.check(y, want[0], want[1], "prompt")
    pages, ck, cv = (t.cuda() for t in cache_of(5, [L], page, H * D, dt))
    lengths = torch.tensor([L], dtype=torch.int32, device="cuda")
    ca.paged_append_(ck, cv, k[0].cuda(), v[0].cuda(), pages, lengths, offsets=torch.tensor([0, L], dtype=torch.int32, device="cuda"))
    for n in (1, 200):
        offsets = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        y = ca.paged_mh_attention(q[0, L - n:].cuda(), ck, cv, pages, lengths, None, H, offsets=offsets, **dev)
        M.check(y, want[0][0, L - n:], want[1][0, L - n:], f"{n} tokens")


@pytest.mark.parametrize("shape", [(1, 666, 1, 8, 181, 20.0, 3), (1, 900, 2, 64, None, 7.0, None)], ids=str)
def test_float32_signals_keep_their_precision(ca, shape):
    """Gradients of capped scores (2-norm): a product's exponent is rounded by 2^-24 of its
    size, which is the largest capped score times log2(e), 29, and twice that with the sum
    of the weights; sums of n terms add sqrt(n) 2^-24.  Results of those are off by less than
    2^-19 of themselves: (2 * 29 ln 2 + sqrt(900)) 2^-24 = 70 * 2^-24 at most, and a
    quarter as rounding errors are not all alike."""
    B, L, H, D, W, cap, docs = shape
    q, k, v, dy = (randn(90 + i, B, L, H * D, scale=3.0 if i == 0 else 1.0) for i in range(4))
    kw = {"cap": cap, "places": None if docs is None else places_of([[docs] * (L // docs)], L)}
    got = run(ca, q, k, v, dy, W or L, H, H, 0, None, kw)
    want = M.sliding(*(t.double() for t in (q, k, v)), W or L, H, H, 0, 1 / math.sqrt(D), None, torch.float32, dy=dy.double(), **kw)
    for g, (x, _), name in zip(got, want, ("y", "dq", "dk", "dv")):
        assert float((g.detach().double().cpu() - x).norm() / x.norm()) <= 70 * 2.0 ** -26, name


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(2, 5, 14, 2, 8), (1, 4, 16, 4, 128), (2, 2, 5, 1, 128), (1, 120, 2, 2, 64)], ids=str)
def test_gradients_of_short_signals(ca, shape, dtype):
    """Weights and score gradients go into the keys' gradients in two values, so that these
    are off by their own rounding e (2-norm) and little more; <dy, y> with the weights'
    rounding in y, as in test_query_gradients_of_few_keys, adds at most e to dk's."""
    B, L, H, Hk, D = shape
    q, k, v, dy = (randn(95 + i, B, L, h * D, dtype=DT[dtype], scale=3.0 if i == 0 else 1.0) for i, h in enumerate((H, Hk, Hk, H)))
    kw = {"cap": 21.0}
    got = run(ca, q, k, v, dy, L, H, Hk, 0, None, kw)
    want = M.sliding(*(t.double() for t in (q, k, v)), L, H, Hk, 0, 1 / math.sqrt(D), None, DT[dtype], dy=dy.double(), **kw)
    for g, (x, _) in zip(got[1:], want[1:]):
        e = float((x.to(DT[dtype]).double() - x).norm())
        assert float((g.double().cpu() - x).norm()) <= math.sqrt(2.0) * e



@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S,W", [(1, 1), (4, 30), (130, 2)], ids=str)
def test_sinks_of_signals_without_their_prefix(ca, S, W, dtype):
    """A batch whose prefixes are empty but for one: sinks are seen from behind the windows
    of their keys' blocks all the same."""
    compare(ca, 3, 420, 2, 1, 32, W, S, (420, 420, 300), DT[dtype],
            {"cap": 15.0, "prefix": torch.tensor([3, 0, 0], dtype=torch.int32)})



@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("W,docs", [(3, None), (40, None), (None, 30)], ids=str)
def test_query_gradients_of_few_keys(ca, W, docs, dtype):
    """Where few keys carry a row its score gradients cancel.  Rounded results alone are
    off by a number e of the type (2-norm).  On top of those come weights rounded in y,
    normalised by their own sum: with n keys that carry a row, the part of their
    errors (e each) along the row's mean falls away, and what is left in <dy, y> is at
    most e times the spread of <dy, v> over the row, the size of the score gradients
    themselves.  Both together: sqrt(2) e."""
    L, H, D = 400, 2, 64
    q, k, v, dy = (randn(60 + i, 1, L, H * D, dtype=DT[dtype], scale=3.0 if i == 0 else 1.0) for i in range(4))
    shape = {"cap": 30.0, "places": None if docs is None else places_of([[docs] * (L // docs)], L)}
    got = run(ca, q, k, v, dy, W, H, H, 0, None, shape)
    want = M.sliding(*(t.double() for t in (q, k, v)), W or L, H, H, 0, 1 / math.sqrt(D), None, DT[dtype], dy=dy.double(), **shape)
    exact = want[1][0]
    e = float((exact.to(DT[dtype]).double() - exact).norm())
    assert float((got[1].double().cpu() - exact).norm()) <= math.sqrt(2.0) * e



def test_slopes_with_a_tangent_are_refused(ca):
    import torch.autograd.forward_ad as fwAD
    q = torch.zeros(1, 8, 32, device="cuda")
    with fwAD.dual_level():
        slopes = fwAD.make_dual(torch.ones(2, device="cuda"), torch.ones(2, device="cuda"))
        with pytest.raises((RuntimeError, NotImplementedError)):
            ca.sliding_mh_attention(q, q, q, None, 2, slopes=slopes)


def test_arrays_written_before_the_backward_are_noticed(ca):
    q, k, v = (randn(3 + i, 1, 40, 64).cuda().requires_grad_(True) for i in range(3))
    for name, t in (("slopes", torch.ones(2, device="cuda")), ("prefix", torch.tensor([5], dtype=torch.int32, device="cuda")),
                    ("places", torch.arange(40, dtype=torch.int32, device="cuda")[None].clone())):
        y = ca.sliding_mh_attention(q, k, v, 10, 2, **{name: t})
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_slopes_far_out(ca):
    """Distances whose bias passes what exponentials hold: the far keys count nothing."""
    L, H, D = 4000, 2, 32
    q, k, v, dy = (randn(5 + i, 1, L, H * D, dtype=torch.bfloat16) for i in range(4))
    slopes = torch.tensor([5.0, 0.0])
    got = run(ca, q, k, v, dy, None, H, H, 0, None, {"slopes": slopes})
    for g in got:
        assert torch.isfinite(g).all()
    want = M.sliding(*(t.double() for t in (q, k, v)), L, H, H, 0, 1 / math.sqrt(D), None, torch.bfloat16, slopes=slopes)
    M.check(got[0], *want[0], "y")


def test_places_that_are_not_ascending_stay_in_bounds(ca):
    """Numbers of any kind: rows may hold anything, but the call ends as others do."""
    L = 300
    q, k, v, dy = (randn(5 + i, 2, L, h * 32, dtype=torch.bfloat16) for i, h in enumerate((2, 1, 1, 2)))
    r = torch.Generator().manual_seed(1)
    for places in (torch.randint(-2 ** 31, 2 ** 31 - 1, (2, L), generator=r).int(),
                   torch.full((2, L), -2 ** 31, dtype=torch.int32), torch.full((2, L), 2 ** 31 - 1, dtype=torch.int32),
                   torch.randint(0, L, (2, L), generator=r).int()):
        for W, S in ((None, 0), (20, 30)):
            got = run(ca, q, k, v, dy, W, 2, 1, S, torch.tensor([300, 77], dtype=torch.int32), {"places": places, "cap": 9.0})
            assert all((g[1, 77:] == 0).all() for g in got)


@pytest.mark.parametrize("D,W", [(64, None), (32, 40)], ids=str)
def test_places_behind_the_lengths_are_not_looked_at(ca, D, W):
    L, H, lens = 900, 2, (900, 111, 300)
    q, k, v, dy = (randn(80 + i, 3, L, H * D, dtype=torch.bfloat16) for i in range(4))
    places = places_of([[60, 200, 5, 700], [70, 1000], [130, 128, 1000]], L)
    lengths = torch.tensor(lens, dtype=torch.int32)
    want = run(ca, q, k, v, dy, W or L, H, H, 3, lengths, {"places": places})
    g = torch.Generator().manual_seed(1)
    for low, high in ((-5, 5), (-2 ** 31, 2 ** 31 - 1), (L, 2 * L)):
        other = places.clone()
        for b, n in enumerate(lens):
            other[b, n:] = torch.randint(low, high, (L - n,), generator=g, dtype=torch.int64).int()
        for a, b in zip(run(ca, q, k, v, dy, W or L, H, H, 3, lengths, {"places": other}), want):
            assert torch.equal(a, b)



def test_rows_apart_streams_and_graphs(ca):
    """Parts of one projection read in place, on a stream of their own, and captured with the
    backward: every replay gives the eager results."""
    B, L, H, Hk, D = 2, 300, 4, 2, 64
    dt = torch.bfloat16
    qkv = randn(3, B, L, (H + 2 * Hk) * D, dtype=dt).cuda()
    slopes, prefix = geometric(H).cuda(), torch.tensor([70, 5], dtype=torch.int32, device="cuda")
    kw = dict(kv_heads=Hk, sinks=3, cap=20.0, slopes=slopes, prefix=prefix)
    dy = randn(4, B, L, H * D, dtype=dt).cuda()

    def step(x):
        x = x.detach().requires_grad_(True)
        q, k, v = x.split([H * D, Hk * D, Hk * D], -1)
        y = ca.sliding_mh_attention(q, k, v, 100, H, **kw)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    eager = step(qkv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(qkv)
        static = qkv.clone()
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(3):
        fresh = randn(60 + i, *qkv.shape, dtype=dt).cuda()
        prefix.copy_(torch.tensor([9 * i, 300 - i], dtype=torch.int32))
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(step(fresh), out):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
def cache_of(seed, lens, page, Ck, dt, extra=3):
    need = [-(-n // page) for n in lens]
    order = list(range(sum(need) + extra))
    random.Random(seed).shuffle(order)
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (max(need + [1]) - n))
        at += n
    k, v = (randn(seed + i, len(order), page, Ck, dtype=dt) for i in (1, 2))
    return torch.tensor(rows, dtype=torch.int32), k, v


PAGED = [
    # H, Hk, D, W, S, page, lengths, new
    (4, 2, 64, None, 0, 16, [1], [1]),
    (8, 2, 64, 30, 5, 16, [1, 77, 300, 16], [1, 1, 1, 1]),
    (5, 5, 40, None, 0, 8, [90, 31, 0, 64], [1, 1, 1, 1]),
    (6, 2, 80, 50, 3, 32, [150, 71, 33], [40, 1, 33]),
    (4, 1, 104, 65, 70, 64, [333, 200], [333, 129]),
    (32, 4, 128, 500, 0, 16, [900, 64], [70, 64]),
    (2, 2, 24, 3, 130, 128, [700], [100]),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["cap", "slopes", "prefix", "all"])
@pytest.mark.parametrize("shape", PAGED, ids=str)
def test_paged(ca, shape, kind, dtype):
    H, Hk, D, W, S, page, lens, new = shape
    dt = DT[dtype]
    print("paged", shape, kind, dtype, flush=True)
    pages, ck, cv = cache_of(5, lens, page, Hk * D, dt)
    offs = [0]
    for n in new:
        offs.append(offs[-1] + n)
    q = randn(9, offs[-1], H * D, dtype=dt, scale=3.0)
    sh = {}
    if kind in ("cap", "all"):
        sh["cap"] = 12.0
    if kind in ("slopes", "all"):
        sh["slopes"] = geometric(H)
    if kind in ("prefix", "all"):
        sh["prefix"] = torch.tensor([(3 * n) // 4 + 1 for n in lens], dtype=torch.int32)
    offsets = torch.tensor(offs, dtype=torch.int32)
    one = all(n == 1 for n in new)
    got = ca.paged_mh_attention(q.cuda(), ck.cuda(), cv.cuda(), pages.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), W, H,
                                kv_heads=Hk, sinks=S, offsets=None if one else offsets.cuda(),
                                **{n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in sh.items()})
    want = M.paged(q.double(), ck.double(), cv.double(), pages, lens, offs, W or 1 << 30, H, Hk, S, 1 / math.sqrt(D), dt, **sh)
    M.check(got, *want, "y")


@pytest.mark.parametrize("one", [True, False])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_paged_pages_outside_the_cache_and_bad_values_behind(ca, one, value):
    """Pages that are not there hide their tokens, of a prefix too; a value that is not
    finite reaches the rows that see it alone; rows that see nothing are zero."""
    H, Hk, D, page, W, dt = 4, 2, 64, 16, 20, torch.bfloat16
    lens, new = [100, 60, 40], [1, 1, 1] if one else [9, 40, 40]
    pages, ck, cv = cache_of(7, lens, page, Hk * D, dt)
    pages[0, 1], pages[1, :] = 10 ** 6, -1
    cv[pages[2, 0].item(), 3] = value
    offs = [0]
    for n in new:
        offs.append(offs[-1] + n)
    q = randn(9, offs[-1], H * D, dtype=dt)
    prefix = torch.tensor([30, 50, 2], dtype=torch.int32)
    sh = {"cap": 9.0, "slopes": geometric(H), "prefix": prefix}
    got = ca.paged_mh_attention(q.cuda(), ck.cuda(), cv.cuda(), pages.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), W, H,
                                kv_heads=Hk, offsets=None if one else torch.tensor(offs, dtype=torch.int32).cuda(),
                                **{n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in sh.items()}).cpu()
    clean = torch.where(torch.isfinite(cv), cv, torch.zeros_like(cv))
    y, by = M.paged(q.double(), ck.double(), clean.double(), pages, lens, offs, W, H, Hk, 0, 1 / math.sqrt(D), dt, **sh)
    sees = torch.zeros(offs[-1], dtype=torch.bool)
    pos = torch.arange(lens[2] - new[2], lens[2])
    sees[offs[2]:] = (pos >= 3) & (pos - 3 < W)
    M.check(got[~sees], y[~sees], by[~sees], "rows that do not see it")
    assert not torch.isfinite(got[sees]).any()
    assert (got[offs[1]:offs[2]] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_serving_gives_the_rows_of_the_whole(ca, dtype):
    """A signal in pieces over a cache: the rows of the whole, for every shape that both take."""
    H, Hk, D, L, page, W, S = 4, 2, 64, 150, 16, 40, 3
    dt = DT[dtype]
    q, k, v = (randn(3 + i, 1, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk)))
    for sh in ({"cap": 10.0}, {"slopes": geometric(H)}, {"cap": 10.0, "slopes": geometric(H), "prefix": torch.tensor([50], dtype=torch.int32)}):
        dev = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in sh.items()}
        pages, ck, cv = (t.cuda() for t in cache_of(5, [L], page, Hk * D, dt))
        got, at = [], 0
        for n in (70, 1, 1, 40, 38):
            at += n
            lengths = torch.tensor([at], dtype=torch.int32, device="cuda")
            offsets = torch.tensor([0, n], dtype=torch.int32, device="cuda")
            ca.paged_append_(ck, cv, k[0, at - n:at].cuda(), v[0, at - n:at].cuda(), pages, lengths, offsets=offsets)
            got.append(ca.paged_mh_attention(q[0, at - n:at].cuda(), ck, cv, pages, lengths, W, H, kv_heads=Hk, sinks=S,
                                             offsets=offsets, **dev))
        want = M.sliding(*(t.double() for t in (q, k, v)), W, H, Hk, S, 1 / math.sqrt(D), None, dt, **sh)[0]
        M.check(torch.cat(got), want[0][0], want[1][0], "y")


def test_paged_captured_follows_its_arrays(ca):
    H, Hk, D, page, dt = 8, 2, 128, 16, torch.bfloat16
    lens = [500, 33, 260]
    pages, ck, cv = (t.cuda() for t in cache_of(5, lens, page, Hk * D, dt))
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    prefix = torch.tensor([10, 20, 30], dtype=torch.int32, device="cuda")
    slopes = geometric(H).cuda()
    q = randn(1, 3, H * D, dtype=dt).cuda()

    def call():
        return ca.paged_mh_attention(q, ck, cv, pages, lengths, 64, H, kv_heads=Hk, cap=15.0, slopes=slopes, prefix=prefix)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        q.copy_(randn(70 + i, 3, H * D, dtype=dt))
        lengths.copy_(torch.tensor([500 - 100 * i, 33 - i, 200 + i], dtype=torch.int32))
        prefix.copy_(torch.tensor([100 * i, 0, 260], dtype=torch.int32))
        slopes.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def plain_block(m, x, places=None, prefix=None):
    """SlidingAttBlock in Float64 on the CPU."""
    w = {n: p.detach().double().cpu() for n, p in m.named_parameters()}
    xd = x.detach().double().cpu()
    qkv = xd @ w["qkv.weight"].T + w["qkv.bias"]
    q, k, v = qkv.split(m.parts, -1)
    D = m.parts[0] // m.nheads
    y = M.sliding(q, k, v, m.window, m.nheads, m.kv_heads, m.sinks, 1 / math.sqrt(D), None, torch.float32, cap=m.cap or 0.0,
                  slopes=None if m.slopes is None else m.slopes.cpu(), places=places, prefix=prefix)[0][0]
    return xd + y @ w["o.weight"].T + w["o.bias"]


def test_block_trains_and_serves(ca):
    """SlidingAttBlock with a cap and a bias by distance: documents, a prefix, a step over a
    cache; its gradients against differences of the 64-bit form."""
    torch.manual_seed(0)
    C, L, page = 64, 60, 8
    m = ca.SlidingAttBlock(C, 16, nheads=4, kv_heads=2, sinks=2, cap=2.0, distance=True).cuda()
    assert m.slopes.dtype == torch.float32 and "slopes" not in m.state_dict()
    x = randn(400, 2, L, C)
    places = places_of([[25, 35], [3, 40, 17]], L)
    prefix = torch.tensor([20, 33], dtype=torch.int32)
    w = randn(401, 2, L, C)
    for kw in ({}, {"places": places}, {"prefix": prefix}):
        xg = x.cuda().requires_grad_(True)
        y = m(xg, **{n: t.cuda() for n, t in kw.items()})
        want = plain_block(m, x, **kw)
        # Float32 projections of 64 channels around the attention: 3 * 64 products' roundings
        tol = 400 * 2.0 ** -24 * float(want.abs().max() + 4)
        assert float((y.detach().double().cpu() - want).abs().max()) <= tol
        (g,) = torch.autograd.grad(y, xg, w.cuda())
        d, h = randn(402, 2, L, C), 2.0 ** -8
        slope = [float(((plain_block(m, x + s * h * d, **kw) - plain_block(m, x - s * h * d, **kw)) * w.double()).sum())
                 / (2 * s * h) for s in (1, 2)]
        assert abs(float((g.double().cpu() * d).sum()) - slope[0]) <= (abs(slope[0] - slope[1])
                                                                      + 400 * 2.0 ** -24 * float(w.abs().sum() * 4))
    ck, cv = (torch.full((20, page, 32), math.nan, device="cuda") for _ in range(2))
    pages = torch.arange(16, dtype=torch.int32).flip(0).reshape(2, 8).contiguous().cuda()
    n = 40
    offs = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    xs = x.cuda()
    full = lambda i: torch.full((2,), i, dtype=torch.int32, device="cuda")
    out = m.step(xs[:, :n].reshape(2 * n, C), ck, cv, pages, full(n), offs, prefix=prefix.cuda())
    assert float((out.reshape(2, n, C).double().cpu() - want[:, :n]).abs().max()) <= tol
    for i in range(n, L):
        out = m.step(xs[:, i], ck, cv, pages, full(i + 1), prefix=prefix.cuda())
        assert float((out.double().cpu() - want[:, i]).abs().max()) <= tol, i
    half = m.to(torch.bfloat16)
    assert half.slopes.dtype == torch.float32 and half(xs.bfloat16()).dtype == torch.bfloat16


def test_positions_count_from_each_document(ca):
    """A block with rotary positions and places turns each document from its own start."""
    torch.manual_seed(3)
    m = ca.SlidingAttBlock(64, 20, nheads=2, rotary=(8,)).cuda()
    x = randn(5, 1, 50, 64).cuda()
    places = places_of([[20, 30]], 50).cuda()
    y = m(x, places=places)
    apart = torch.cat([m(x[:, :20]), m(x[:, 20:])], 1)
    assert float((y - apart).detach().abs().max()) <= 400 * 2.0 ** -24 * float(apart.detach().abs().max() + 4)


def test_refusals_on_device_tensors(ca):
    x = torch.zeros(2, 8, 64, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    q, cache, table, one = x[0], torch.zeros(4, 8, 64, device="cuda"), torch.zeros((8, 2), **i32), torch.ones(8, **i32)
    held, n = torch.zeros(4, **i32), torch.zeros(8, **i32)
    cases = [
        (AssertionError, "cap", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, cap=-1.0)),
        (AssertionError, "cap", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, cap=1e35)),
        (AssertionError, "slopes", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, slopes=torch.zeros(3, device="cuda"))),
        (AssertionError, "device", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, slopes=torch.zeros(2))),
        (AssertionError, "gradients", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, slopes=torch.zeros(2, device="cuda", requires_grad=True))),
        (AssertionError, "shape", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, prefix=torch.zeros(3, **i32))),
        (AssertionError, "shape", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, places=torch.zeros(8, **i32))),
        (AssertionError, "together", lambda: ca.sliding_mh_attention(x, x, x, 3, 2, prefix=torch.zeros(2, **i32), places=torch.zeros((2, 8), **i32))),
        (AssertionError, "slopes", lambda: ca.paged_mh_attention(q, cache, cache, table, one, 3, 2, slopes=torch.zeros(1, device="cuda"))),
        (AssertionError, "prefix", lambda: ca.paged_mh_attention(q, cache, cache, table, one, 3, 2, prefix=torch.zeros(2, **i32))),
        (AssertionError, "counts", lambda: ca.paged_compact_(cache, cache, table, torch.zeros(3, **i32))),
        (AssertionError, "to must have", lambda: ca.paged_resize_(cache, cache, table, n, held, n[:3])),
        (AssertionError, "strides", lambda: ca.paged_resize_(cache, torch.zeros(4, 8, 128, device="cuda")[..., :64], table, n, held, n)),
        (TypeError, "counts", lambda: ca.paged_fork(table, n, None, n, 8)),
        (TypeError, "source", lambda: ca.paged_fork(table, n, held, table, 8)),
        (NotImplementedError, "power of two", lambda: ca.paged_fork(table, n, held, n, 12)),
        (AssertionError, "device", lambda: ca.paged_resize_(cache, cache, table, n, held, n.cpu())),
        (AssertionError, "lengths must have", lambda: ca.paged_fork(table, n[:2], held, n, 8)),
    ]
    for kind, text, call in cases:
        with pytest.raises(kind, match=text):
            call()
