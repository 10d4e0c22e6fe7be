"""sliding_mh_attention's gradients in each plan of the keys' pass, against the
64-bit restatement within its bounds."""
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


# B, L, H, Hk, D, W, S: one workgroup a block of 128 keys, and up to four groups of 32
# sinks that rows behind the block's window see
ONE_PART = [
    (8, 512, 8, 8, 32, 64, 130),
    (8, 512, 8, 8, 64, 64, 130),
    (4, 512, 16, 16, 96, 64, 130),
    (8, 512, 8, 8, 128, 64, 130),
    (2, 512, 64, 32, 128, 64, 100),
    (1, 1024, 64, 32, 64, 200, 70),
    (4, 300, 32, 32, 40, 20, 280),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", ONE_PART, ids=str)
def test_far_sinks_without_a_join(ca, shape, dtype):
    B, L, H, Hk, D, W, S = shape
    dt = DT[dtype]
    parts, far, _, _ = walk_split(*shape, dt)
    assert parts == 1 and far >= 3
    print("one part", shape, dtype, flush=True)
    q, k, v, dy = (randn(7 + i, B, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H)))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=Hk, sinks=S)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    want = M.sliding(*(t.double() for t in (q, k, v)), W, H, Hk, S, 1 / math.sqrt(D), None, dt, dy.double())
    for got, (x, bx), name in zip((y, *grads), want, ("y", "dq", "dk", "dv")):
        M.check(got, x, bx, name)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("shape", [(2, 200, 4, 2, 64, 30, 3), (8, 512, 8, 8, 64, 64, 40)], ids=str)
def test_padding_gets_no_gradient_from_a_bad_row(ca, shape, value, dtype):
    """A row of q, dy, k or v that is not finite, in the last token of a signal:
    gradients behind the signal's length are zeros all the same."""
    B, L, H, Hk, D, W, S = shape
    dt = DT[dtype]
    assert (walk_split(*shape, dt)[0] == 1) == (B == 8)
    lens = torch.tensor([L - 37 - b for b in range(B)], dtype=torch.int32)
    base = [randn(17 + i, B, L, h * D, dtype=dt) for i, h in enumerate((H, Hk, Hk, H))]
    for which in range(4):
        t = [x.clone() for x in base]
        for b in range(B):
            t[which][b, int(lens[b]) - 1, ::3] = value
        leaves = [x.cuda().requires_grad_(True) for x in t[:3]]
        y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=Hk, sinks=S, lengths=lens.cuda())
        for x in (y, *torch.autograd.grad(y, leaves, t[3].cuda())):
            for b in range(B):
                assert (x[b, int(lens[b]):] == 0).all(), which
