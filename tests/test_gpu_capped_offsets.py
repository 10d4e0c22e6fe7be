"""Capped scores that are all far below zero: under the softmax's fixed reference (BFloat16, caps
to 62) weights are as small as 2^-80 then.  Right against 64 bits, whatever the size of the
values, and as fast as other scores: rows are not formed again one by one for it."""
import math
import time

import pytest
import torch

import shaped_model as M

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def low(seed, n, H, Hk, D, offset, dtype, size=1.0):
    """q, k, v, dy of (1, n, heads * D) whose scores lie about `offset` before the cap (scale 1/sqrt(D)): one
    channel carries it; values of some size."""
    g = torch.Generator().manual_seed(seed)
    q, k, v, dy = (torch.randn((1, n, h, D), generator=g) for h in (H, Hk, Hk, H))
    a = math.sqrt(abs(offset) * math.sqrt(D))
    q[..., 0], k[..., 0] = a, math.copysign(a, offset)
    return [t.reshape(1, n, -1).to(dtype) for t in (q, k, v * size, dy)]


@pytest.mark.parametrize("dtype,size", [("bf16", 1.0), ("bf16", 1e-20), ("bf16", 1e-30), ("bf16", 1e25), ("f16", 1.0), ("f32", 1.0)])
@pytest.mark.parametrize("cap,offset", [(30.0, -60), (50.0, -55), (50.0, -300), (60.0, -40), (62.0, -1000)])
def test_low_scores(ca, dtype, size, cap, offset):
    dt, n, H, Hk, D = DT[dtype], 200, 4, 2, 64
    q, k, v, dy = low(3, n, H, Hk, D, offset, dt, size)
    if size > 1:
        dy = dy * 2.0 ** -90  # (so that Float32 holds <dy, y> and the gradients)
    for W, shape in ((n, {}), (40, {}), (60, {"prefix": torch.tensor([30], dtype=torch.int32)}),
                     (n, {"places": torch.tensor([list(range(70)) + list(range(n - 70))], dtype=torch.int32)})):
        leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=Hk, cap=cap, **{s: t.cuda() for s, t in shape.items()})
        got = (y, *torch.autograd.grad(y, leaves, dy.cuda()))
        want = M.sliding(q.double(), k.double(), v.double(), W, H, Hk, 0, 1 / math.sqrt(D), None, dt, cap=cap, dy=dy.double(), **shape)
        for a, (x, bx), name in zip(got, want, ("y", "dq", "dk", "dv")):
            M.check(a.detach().cpu(), x, bx, f"{name}, window {W}")


@pytest.mark.parametrize("dtype,size", [("bf16", 1.0), ("bf16", 1e-30), ("f16", 1.0), ("f32", 1.0)])
@pytest.mark.parametrize("cap,offset", [(50.0, -55), (62.0, -1000)])
@pytest.mark.parametrize("new", [1, 9, 150])
def test_low_scores_over_a_cache(ca, dtype, size, cap, offset, new):
    dt, n, H, Hk, D, page = DT[dtype], 400, 4, 2, 64, 16
    q, k, v, _ = low(4, n, H, Hk, D, offset, dt, size)
    q, caches = q[0, n - new:], [t.reshape(n // page, page, Hk * D) for t in (k, v)]
    pages, lens, offs = torch.arange(n // page, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32), torch.tensor([0, new], dtype=torch.int32)
    for W in (n, 20):
        y = ca.paged_mh_attention(q.cuda(), *(t.cuda() for t in caches), pages.cuda(), lens.cuda(), W, H, kv_heads=Hk, cap=cap,
                                  offsets=offs.cuda())
        x, bx = M.paged(q.double(), *(t.double() for t in caches), pages, lens, offs, W, H, Hk, 0, 1 / math.sqrt(D), dt, cap=cap)
        M.check(y.cpu(), x, bx, f"window {W}")


def test_time_of_low_scores(ca):
    """2048 tokens, 32 heads of 128 over 8, cap 60, scores about -40: 0.08 ms as others, 5.9 where every
    row is formed again."""
    n, H, Hk, D = 2048, 32, 8, 128
    q, k, v = (t.cuda() for t in low(5, n, H, Hk, D, -40, torch.bfloat16)[:3])

    def call():
        return ca.sliding_mh_attention(q, k, v, n, H, kv_heads=Hk, cap=60.0)

    call()
    least = math.inf
    for _ in range(5):
        torch.cuda.synchronize()
        t = time.perf_counter()
        call()
        torch.cuda.synchronize()
        least = min(least, time.perf_counter() - t)
    assert least < 2e-3, least
