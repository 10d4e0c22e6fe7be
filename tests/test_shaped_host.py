"""Refusals of the shaped token attention and of the cache's pages, on the CPU: the C
ABI's argument checks, which precede every launch, and the Python layer's.  No kernel
runs."""
import ctypes
import math
import random

import pytest
import torch

import pages_model as PM

P = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first
FAR = ctypes.c_void_p(0x7000000000)
FAR2 = ctypes.c_void_p(0x7100000000)
FAR3 = ctypes.c_void_p(0x7200000000)
FAR4 = ctypes.c_void_p(0x7300000000)
ODD = ctypes.c_void_p(0x10008)


@pytest.fixture(scope="module")
def L():
    from circulant_attention import _lib
    return _lib


def expect(L, rc, code, fragment):
    assert rc == code, (rc, L.lib.circatt_last_error())
    assert fragment in L.lib.circatt_last_error().decode(), L.lib.circatt_last_error()


def shape(cap=0.0, slopes=None, prefix=None, places=None, row=0):
    return cap, slopes, prefix, places, row


def fwd(L, sh=shape(), dtype=3, n=64, B=2, H=4, Hk=2, dh=64, W=16, S=0, scale=0.125, q=P, k=P, y=FAR):
    return L.lib.circatt_shaped_fwd(dtype, n, B, H, Hk, dh, W, S, scale, *sh, q, H * dh, 0, k, Hk * dh, 0, P, Hk * dh, 0,
                                    None, y, None, None, None)


def bwd(L, sh=shape(), work=FAR2, wbytes=1 << 32, n=64, dq=FAR, dk=FAR3, dv=FAR4):
    return L.lib.circatt_shaped_bwd(3, n, 2, 4, 2, 64, 16, 0, 0.125, *sh, P, 256, 0, P, 128, 0, P, 128, 0, None, P, None, P, P,
                                    256, 0, dq, dk, dv, work, wbytes, None)


SHAPES = [
    (shape(cap=-1.0), -1, "cap"), (shape(cap=math.nan), -1, "cap"), (shape(cap=math.inf), -1, "cap"),
    (shape(cap=1e-35), -1, "cap"), (shape(cap=1e35), -1, "cap"),
    (shape(prefix=P, places=P, row=64), -1, "do not go together"), (shape(places=P, row=-1), -1, "negative stride"),
]


@pytest.mark.parametrize("sh,code,fragment", SHAPES)
def test_shapes(L, sh, code, fragment):
    expect(L, fwd(L, sh), code, fragment)
    expect(L, bwd(L, sh), code, fragment)
    if sh[3] is None:
        expect(L, paged(L, sh[:3]), code, fragment)


def test_lengths_that_slopes_do_not_count(L):
    expect(L, fwd(L, shape(slopes=P), n=(1 << 24) + 1), -2, "2^24")
    expect(L, bwd(L, shape(slopes=P), n=(1 << 24) + 1), -2, "2^24")
    expect(L, paged(L, (0.0, P, None), maxp=1 << 21, page=16), -2, "2^24")


@pytest.mark.parametrize("args,code,fragment", [
    (dict(dtype=1), -2, "dtype"), (dict(H=4, Hk=3), -1, "divisible by kv_heads"), (dict(dh=12), -2, "multiple of 8"),
    (dict(W=0), -1, "window"), (dict(scale=0.0), -1, "scale"), (dict(q=None), -1, "q is NULL"), (dict(q=ODD), -1, "16-byte"),
    (dict(y=None), -1, "y is NULL"), (dict(k=FAR), -1, "y must not overlap k"), (dict(n=1 << 20, B=1 << 12), -2, "2^31"),
])
def test_sliding_arguments(L, args, code, fragment):
    expect(L, fwd(L, shape(cap=20.0), **args), code, fragment)


def test_results_stay_off_the_shape(L):
    for sh, name in ((shape(slopes=FAR), "slopes"), (shape(prefix=FAR), "prefix"), (shape(places=FAR, row=64), "places")):
        expect(L, fwd(L, sh), -1, f"y must not overlap {name}")
        expect(L, bwd(L, sh), -1, f"dq must not overlap {name}")
    # the last of the places
    expect(L, fwd(L, shape(places=ctypes.c_void_p(FAR.value - 4 * (1000 + 63)), row=1000)), -1, "y must not overlap places")
    for sh, name in (((0.0, FAR, None), "slopes"), ((0.0, None, FAR), "prefix")):
        expect(L, paged(L, sh), -1, f"y must not overlap {name}")


def test_nothing_to_do(L):
    assert fwd(L, shape(cap=3.0), n=0, q=None) == 0
    assert fwd(L, shape(cap=3.0), B=0, q=None) == 0
    expect(L, fwd(L, shape(cap=-3.0), n=0), -1, "cap")
    assert paged(L, (3.0, None, None), T=0, B=1, offsets=P) == 0


def test_workspaces(L):
    size, plain = L.lib.circatt_shaped_bwd_workspace_bytes, L.lib.circatt_sliding_bwd_workspace_bytes
    args = (3, 500, 2, 4, 2, 64, 16, 0)
    assert size(*args, 0, 0) >= plain(*args)
    assert size(*args, 1, 0) >= size(*args, 0, 0) + 4 * (500 * 4 + 500 * 2)  # slopes and tokens of packed rows
    assert size(*args, 0, 1) >= 4 * (500 * 4 * 2 + 500 * 2)                  # sums of the rows, ends of documents
    # sinks behind the window are a walk of their own, but not with documents or a prefix
    far = (3, 4000, 2, 4, 2, 64, 16, 40)
    assert size(*far, 0, 0) > size(*far, 0, 1)
    assert size(*args, 0, 3) == size(*args, 0, -1) == -1
    assert size(3, 0, 2, 4, 2, 64, 16, 0, 1, 1) == 0 and size(3, 64, 2, 4, 3, 64, 16, 0, 0, 0) == -1
    expect(L, bwd(L, shape(slopes=P), wbytes=100), -1, "workspace of 100")
    expect(L, bwd(L, shape(cap=3.0), work=None), -1, "workspace is NULL")


def paged(L, sh=(0.0, None, None), T=2, B=2, dh=64, page=16, npages=100, maxp=8, offsets=None, y=FAR, work=P, wbytes=1 << 40):
    return L.lib.circatt_shaped_paged(3, T, B, 4, 2, dh, 16, 0, 0.125, *sh, P, 256, P, P, npages, page, page * 128, 128, P, maxp,
                                      maxp, P, offsets, y, 1, work, wbytes, None)


@pytest.mark.parametrize("args,code,fragment", [
    (dict(page=12), -2, "power of two"), (dict(T=3), -1, "one row for each sequence"), (dict(y=P), -1, "must not overlap"),
    (dict(npages=0), -1, "a cache of"), (dict(maxp=0), -1, "page table"), (dict(dh=12), -2, "multiple of 8"),
])
def test_paged_arguments(L, args, code, fragment):
    expect(L, paged(L, (20.0, None, None), **args), code, fragment)


# ---------------------------------------------------------------------------
def fork(L, B=4, npages=100, page=16, pages=P, row=8, maxp=8, lengths=P, counts=P, N=4, source=P, op=FAR, ol=FAR2, oc=FAR3):
    return L.lib.circatt_paged_fork(B, npages, page, pages, row, maxp, lengths, counts, N, source, op, ol, oc, None)


def resize(L, dtype=3, C=64, k=P, v=P, npages=100, page=16, ps=1024, rs=64, B=4, pages=P, row=8, maxp=8, lengths=P, counts=P,
           to=P, op=FAR, ol=FAR2, oc=FAR3, work=FAR4, wbytes=1 << 20):
    return L.lib.circatt_paged_resize(dtype, C, k, v, npages, page, ps, rs, B, pages, row, maxp, lengths, counts, to, op, ol, oc,
                                      work, wbytes, None)


def compact(L, dtype=3, C=64, k=P, v=P, npages=100, page=16, ps=1024, rs=64, B=4, pages=P, row=8, maxp=8, counts=P, op=FAR,
            oc=FAR3, work=FAR4, wbytes=1 << 20):
    return L.lib.circatt_paged_compact(dtype, C, k, v, npages, page, ps, rs, B, pages, row, maxp, counts, op, oc, work, wbytes,
                                       None)


TABLES = [
    (dict(B=0), -1, "sequence count"), (dict(B=65536), -1, "sequence count"), (dict(page=24), -2, "power of two"),
    (dict(npages=0), -1, "a cache of"), (dict(npages=1 << 28), -1, "a cache of"), (dict(maxp=0), -1, "page table"),
    (dict(B=65535, maxp=1 << 15, row=1 << 15, page=1), -2, "a table of"), (dict(row=7), -1, "page table"), (dict(maxp=1 << 27, row=1 << 27), -1, "page table"), (dict(pages=None), -1, "pages is NULL"),
    (dict(counts=None), -1, "counts is NULL"), (dict(oc=None), -1, "out_counts is NULL"),
    (dict(op=None), -1, "out_pages is NULL"), (dict(op=P), -1, "out_pages must not overlap pages"),
    (dict(oc=ctypes.c_void_p(P.value + 396)), -1, "out_counts must not overlap"), (dict(oc=FAR), -1, "must not overlap"),
]


@pytest.mark.parametrize("args,code,fragment", TABLES)
def test_tables(L, args, code, fragment):
    for call in (fork, resize, compact):
        expect(L, call(L, **args), code, fragment)


@pytest.mark.parametrize("args,code,fragment", [
    (dict(dtype=1), -2, "dtype"), (dict(C=0), -1, "channel count"), (dict(k=None), -1, "cache is NULL"),
    (dict(v=ODD), -1, "16-byte"), (dict(rs=56), -1, "strides"), (dict(ps=512), -1, "must not overlap"),
    (dict(rs=68), -1, "16-byte"), (dict(work=None), -1, "workspace is NULL"), (dict(wbytes=300), -1, "workspace of 300"),
    (dict(work=ODD), -1, "16-byte"), (dict(work=P), -1, "workspace must not overlap"), (dict(ps=1 << 36), -2, "63 GiB"),
])
def test_caches_of_pages(L, args, code, fragment):
    for call in (resize, compact):
        expect(L, call(L, **args), code, fragment)


def test_forks_and_sizes(L):
    expect(L, fork(L, N=-1), -1, "sequence count")
    expect(L, fork(L, N=65536), -1, "sequence count")
    expect(L, fork(L, source=None), -1, "source is NULL")
    expect(L, fork(L, lengths=None), -1, "lengths is NULL")
    expect(L, fork(L, ol=None), -1, "out_lengths is NULL")
    expect(L, resize(L, lengths=None), -1, "lengths is NULL")
    expect(L, resize(L, to=None), -1, "to is NULL")
    expect(L, resize(L, ol=None), -1, "out_lengths is NULL")
    expect(L, resize(L, ol=P), -1, "out_lengths must not overlap")
    size = L.lib.circatt_paged_resize_workspace_bytes
    assert size(4, 100) >= 4 * 108 and size(0, 100) == -1 and size(4, 0) == -1
    size = L.lib.circatt_paged_compact_workspace_bytes
    assert size(100) >= 4 * 300 and size(0) == -1


# ---------------------------------------------------------------------------
def test_python_layer():
    from circulant_attention import tokens as T
    q = torch.zeros(2, 9, 32)
    ok = torch.zeros(4)
    cap, *arrays, row = T._shape(q, 2, 4, 5, None, None).args()
    assert cap == 5.0 and row == 0 and not any(arrays)
    assert T._shape(q, 2, 4, None, ok, None).args()[1].value == ok.data_ptr()
    for cap in (-1.0, math.nan, math.inf):
        with pytest.raises(AssertionError, match="cap"):
            T._shape(q, 2, 4, cap, None, None)
    with pytest.raises(TypeError, match="slopes"):
        T._shape(q, 2, 4, None, ok.double(), None)
    with pytest.raises(TypeError, match="slopes"):
        T._shape(q, 2, 4, None, [1.0] * 4, None)
    with pytest.raises(AssertionError, match="slopes must have shape"):
        T._shape(q, 2, 8, None, ok, None)
    with pytest.raises(AssertionError, match="slopes must not require"):
        T._shape(q, 2, 4, None, ok.clone().requires_grad_(True), None)
    with torch.no_grad():
        T._shape(q, 2, 4, None, ok.clone().requires_grad_(True), None)
    with pytest.raises(TypeError, match="prefix"):
        T._shape(q, 2, 4, None, None, torch.zeros(2))
    with pytest.raises(AssertionError, match="prefix must have shape"):
        T._shape(q, 2, 4, None, None, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(AssertionError, match="places must have shape"):
        T._shape(q, 2, 4, None, None, None, torch.zeros(9, dtype=torch.int32))
    with pytest.raises(AssertionError, match="do not go together"):
        T._shape(q, 2, 4, None, None, torch.zeros(2, dtype=torch.int32), torch.zeros((2, 9), dtype=torch.int32))
    ints = torch.zeros((2, 3), dtype=torch.int32)
    for call in (lambda: T.paged_fork(ints, ints[:, 0], ints[0], ints[0], 16),
                 lambda: T.paged_resize_(q, q, ints, ints[:, 0], ints[0], ints[0]),
                 lambda: T.paged_compact_(q, q, ints, ints[0])):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    with pytest.raises(TypeError, match="pages"):
        T.paged_fork(ints.long(), ints[:, 0], ints[0], ints[0], 16)


def test_the_model_of_pages_keeps_count():
    """pages_model.py by itself: counts are what the tables hold, and no page is in two
    hands where tokens are written."""
    r = random.Random(1)
    page, npages, most = 4, 60, 9
    rows, lengths, counts = [[-1] * most for _ in range(5)], [0] * 5, [0] * npages

    def checked(rows, lengths, counts):
        held = [0] * npages
        for row, n in zip(rows, lengths):
            has = PM.reach(n, page, most)
            assert all(p >= 0 for p in row[:has]) and all(p == -1 for p in row[has:])
            for p in row[:has]:
                held[p] += 1
        assert held == counts

    for _ in range(60):
        to = [r.choice([-1, 0, n + 1, n + 1, max(0, n - 2), n + 6]) for n in lengths]
        rows, lengths, counts, moves = PM.resize(rows, lengths, counts, to, page)
        checked(rows, lengths, counts)
        source = [r.choice([-1, *range(len(rows))]) for _ in range(r.randint(2, 7))]
        rows, lengths, counts = PM.fork(rows, lengths, counts, source, page)
        checked(rows, lengths, counts)
        rows, counts, moves = PM.compact(rows, counts)
        checked(rows, lengths, counts)
        assert all(c > 0 for c in counts[:sum(x > 0 for x in counts)])


def test_a_block_keeps_its_slopes():
    import circulant_attention as ca

    m = ca.SlidingAttBlock(64, 20, nheads=2, distance=True)
    assert torch.equal(m.slopes, torch.tensor([2.0 ** -4, 2.0 ** -8]))
    m.slopes.mul_(3.0)  # others than it was made with
    m = m.to(torch.bfloat16)
    assert m.slopes.dtype == torch.float32 and torch.equal(m.slopes, 3.0 * torch.tensor([2.0 ** -4, 2.0 ** -8]))
    assert next(m.parameters()).dtype == torch.bfloat16
    m = m.to("meta").to_empty(device="cpu")
    assert torch.equal(m.slopes, torch.tensor([2.0 ** -4, 2.0 ** -8])) and "slopes" not in m.state_dict()
