"""paged_mh_attention of few new tokens behind prefixes that reach far beyond their windows:
blocks of rows whose walks are split into parts by what the prefix makes of them, against the
64-bit restatement of shaped_model.py."""
import ctypes
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


def batch(seed, dtype, lens, new, H, Hk, D, page, spare=2, missing=()):
    """(q, cache_k, cache_v, pages, lengths, offsets) of sequences of lens tokens, new[b] of them new; pages
    in no order, those of `missing` (sequence, entry) not in the cache."""
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    most = max(-(-n // page) for n in lens) + 1
    npages = sum(-(-n // page) for n in lens) + spare
    order = list(range(npages))
    r.shuffle(order)
    rows, at = [], 0
    for n in lens:
        has = -(-n // page)
        rows.append(order[at:at + has] + [-1] * (most - has))
        at += has
    for b, e in missing:
        rows[b][e] = r.choice([-1, npages, -5])
    offs = [0]
    for n in new:
        offs.append(offs[-1] + n)
    q = torch.randn((offs[-1], H * D), generator=g).to(dtype)
    k, v = (torch.randn((npages, page, Hk * D), generator=g).to(dtype) for _ in range(2))
    return q, k, v, torch.tensor(rows, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32), torch.tensor(offs, dtype=torch.int32)


def compare(ca, args, prefix, W, H, Hk, S, dtype, ones, **shape):
    q, k, v, pages, lens, offs = args
    D = q.shape[1] // H
    pf = torch.tensor(prefix, dtype=torch.int32)
    dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in shape.items()}
    y = ca.paged_mh_attention(q.cuda(), k.cuda(), v.cuda(), pages.cuda(), lens.cuda(), W, H, kv_heads=Hk, sinks=S,
                              offsets=None if ones else offs.cuda(), prefix=pf.cuda(), **dev)
    x, bx = M.paged(q.double(), k.double(), v.double(), pages, lens, offs, W, H, Hk, S, D ** -0.5, dtype, prefix=pf, **shape)
    M.check(y.cpu(), x, bx, f"prefixes {prefix}, window {W}")


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("shape", [{}, {"cap": 20.0}, {"cap": 20.0, "slopes": True}])
@pytest.mark.parametrize("H,Hk,D", [(2, 1, 128), (4, 2, 64), (3, 3, 32)])
def test_one_token(ca, dtype, shape, H, Hk, D):
    """Walks of one part beside walks of all, in one launch."""
    shape = dict(shape)
    if shape.pop("slopes", False):
        shape["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1).double() / H).float()
    lens = [2100, 1, 700, 2049, 33]
    args = batch(5, DT[dtype], lens, [1] * 5, H, Hk, D, 16)
    for prefix, W, S in (([2000, 0, 700, 64, 5], 32, 0), ([-3, 1, 100, 1 << 30, 33], 1, 3), ([127, 128, 129, 2048, 32], 700, 0)):
        compare(ca, args, prefix, W, H, Hk, S, DT[dtype], True, **shape)


@pytest.mark.parametrize("dtype", sorted(DT))
def test_few_tokens_each(ca, dtype):
    """Several new tokens: blocks of 32 rows, some of a sequence partly filled."""
    H, Hk, D = 4, 2, 64
    args = batch(6, DT[dtype], [1500, 900, 40], [7, 1, 5], H, Hk, D, 32)
    for prefix, W in (([1400, 0, 38], 16), ([100, 880, 0], 3), ([0, 0, 0], 16)):
        compare(ca, args, prefix, W, H, Hk, 2, DT[dtype], False)


def test_pages_that_are_not_there(ca):
    H, Hk, D = 4, 2, 64
    lens = [1600, 1600]
    args = batch(7, torch.bfloat16, lens, [1, 1], H, Hk, D, 16, missing=[(0, e) for e in range(3, 40)] + [(1, 99)])
    compare(ca, args, [1500, 1500], 8, H, Hk, 0, torch.bfloat16, True)
    compare(ca, args, [640, 10], 8, H, Hk, 0, torch.bfloat16, True, cap=10.0)


def test_values_that_are_not_finite(ca):
    """They reach the heads that see them, and no other sequence."""
    H, Hk, D, dt = 4, 2, 64, torch.bfloat16
    q, k, v, pages, lens, offs = batch(8, dt, [1600, 1600, 1600], [1] * 3, H, Hk, D, 16)
    pf = [1500, 1500, 20]
    v[pages[0, 50], 3, :D] = float("nan")   # seen by sequence 0's first two heads, token 803
    k[pages[2, 50], 3, :] = float("nan")    # behind sequence 2's prefix and before its window: by nobody
    y = ca.paged_mh_attention(q.cuda(), k.cuda(), v.cuda(), pages.cuda(), lens.cuda(), 8, H, kv_heads=Hk,
                              prefix=torch.tensor(pf, dtype=torch.int32, device="cuda")).cpu()
    assert y[0, :2 * D].isnan().all() and not y[0, 2 * D:].isnan().any() and not y[1:].isnan().any()
    fine = [torch.nan_to_num(t) for t in (k, v)]
    x, bx = M.paged(q.double(), *(t.double() for t in fine), pages, lens, offs, 8, H, Hk, 0, D ** -0.5, dt,
                    prefix=torch.tensor(pf))
    M.check(y[1:], x[1:], bx[1:], "the others")
    M.check(y[:1, 2 * D:], x[:1, 2 * D:], bx[:1, 2 * D:], "the other heads")


def test_the_plain_workspace_is_enough(ca):
    """The C entry with what circatt_paged_workspace_bytes asks for (here none): right, by fewer
    workgroups."""
    from circulant_attention import _lib as L
    H, Hk, D, W, page, dt = 4, 2, 64, 8, 16, torch.bfloat16
    q, k, v, pages, lens, offs = batch(9, dt, [1600], [1], H, Hk, D, page)
    most = pages.shape[1]
    room = (L.BF16, 1, 1, H, Hk, D, W, 0, page, most)
    assert L.lib.circatt_paged_workspace_bytes(*room) == 0 == L.lib.circatt_shaped_paged_workspace_bytes(*room, 0)
    need = L.lib.circatt_shaped_paged_workspace_bytes(*room, 1)
    assert need > 0
    t = [x.cuda() for x in (q, k, v, pages, lens, torch.tensor([1500], dtype=torch.int32))]
    x, bx = M.paged(q.double(), k.double(), v.double(), pages, lens, offs, W, H, Hk, 0, D ** -0.5, dt, prefix=torch.tensor([1500]))
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    work = torch.empty(need // 4 + 4, device="cuda")
    for p, nbytes in ((None, 0), (work, need), (work, need - 4), (work[1:], need)):
        y = torch.zeros((1, H * D), dtype=dt, device="cuda")
        L.check(L.lib.circatt_shaped_paged(L.BF16, 1, 1, H, Hk, D, W, 0, D ** -0.5, 0.0, None, t[5].data_ptr(), t[0].data_ptr(), H * D,
                                           t[1].data_ptr(), t[2].data_ptr(), k.shape[0], page, page * Hk * D, Hk * D, t[3].data_ptr(),
                                           most, most, t[4].data_ptr(), None, y.data_ptr(), 1, None if p is None else p.data_ptr(),
                                           nbytes, stream))
        M.check(y.cpu(), x, bx, f"workspace of {nbytes}")


def test_captured_calls_follow_their_prefixes(ca):
    """Parts follow from what the array holds when the kernels run."""
    H, Hk, D, W, dt = 4, 2, 64, 8, torch.bfloat16
    q, k, v, pages, lens, offs = batch(10, dt, [1600, 700], [1, 1], H, Hk, D, 16)
    t = [x.cuda() for x in (q, k, v, pages, lens)]
    pf = torch.zeros(2, dtype=torch.int32, device="cuda")

    def call():
        return ca.paged_mh_attention(*t, W, H, kv_heads=Hk, prefix=pf)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for prefix in ([1600, 0], [0, 690], [1, 1], [900, 300], [0, 0], [1590, 700]):
        pf.copy_(torch.tensor(prefix, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, call())
        x, bx = M.paged(q.double(), k.double(), v.double(), pages, lens, offs, W, H, Hk, 0, D ** -0.5, dt, prefix=torch.tensor(prefix))
        M.check(y.cpu(), x, bx, f"prefixes {prefix}")
