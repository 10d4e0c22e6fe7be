"""Attention on token signals: the sliding window in its causal form with
sinks (the first tokens stay visible), for training and over a paged cache for
serving, its scores capped, biased by distance or masked by documents or a prefix
where that is asked for; the pages of the cache; and rotary positions on one to
three axes.  No counterpart in the reference, whose windows are centred and wrap
around.

Signals are channels-last as in `channels_last=True` of the fused attention:
(B, L, C) with the heads one after another in C.  Float32, Float16 and
BFloat16; heads of a multiple of 8 channels up to 128.  Rows may lie any
distance apart (the parts of one projection's output are read in place).
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib as L
from ._functions import ptr, stream_ptr

_CODES = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}
_EVERY = 1 << 30  # a window that holds every token


def _call(device, fn, *args):
    """fn(*args, stream) on the device's current stream, the device made current
    where it is not."""
    if device.index == torch.cuda.current_device():
        rc = fn(*args, stream_ptr(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream_ptr(device))
    if rc != L.OK:
        L.check(rc)


def _recorded(*tensors):
    """Whether a call goes through its autograd function: one of the tensors
    requires gradients, or forward mode is on, which the function refuses for
    tensors with a tangent."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any([t.requires_grad for t in tensors])


def _require(t, name, like=None, dtypes=_CODES):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on a HIP device (libcircatt has no CPU path)")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise AssertionError(f"{name} must have the type and the device of the first argument")


def _index(t, name, like, shape):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 torch.Tensor")
    if t.device != like.device:
        raise AssertionError(f"{name} must have the type and the device of the first argument")
    if tuple(t.shape) != tuple(shape):
        raise AssertionError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


def _rows(t):
    """(t, row stride, batch stride) of a (B, L, C) signal whose channels are
    adjacent and whose rows are 16-byte aligned; a copy where they are not."""
    B, n, C = t.shape
    sb, sr, sc = t.stride()
    e = 16 // t.element_size()
    if n == 1:
        sr = max(C, (sb if B > 1 and sb >= C else C))
        sr += -sr % e
    if B == 1:
        sb = 0
    if (sc != 1 and C > 1) or sr < C or sr % e or sb % e or t.data_ptr() % 16 or sr > 1 << 22:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        return t, C, C * n
    return t, sr, sb


def _head_count(C, nheads, what):
    if nheads < 1 or C % nheads != 0:
        raise AssertionError(f"{what} channels ({C}) must be divisible by their heads ({nheads})")
    return C // nheads


class _Shape:
    """How a call's scores are shaped: cap (0: none), and slopes, prefix and places or
    None each."""
    __slots__ = ("cap", "arrays", "row")

    def __init__(self, cap, slopes, prefix, places):
        self.cap, self.arrays = cap, (slopes, prefix, places)
        self.row = 0 if places is None else places.shape[1]

    def args(self):
        slopes, prefix, places = self.arrays
        return self.cap, ptr(slopes), ptr(prefix), ptr(places), self.row


def _shape(q, B, nheads, cap, slopes, prefix, places=None):
    """The call's _Shape."""
    cap = float(cap or 0.0)
    if not 0.0 <= cap < math.inf:
        raise AssertionError(f"cap={cap} must be positive and finite, 0 or None: no cap")
    if cap > 0.0 and ctypes.c_float(cap).value == 0.0:
        raise AssertionError(f"cap={cap} is 0 in Float32, in which the kernels take it")
    if prefix is not None and places is not None:
        raise AssertionError("prefix and places do not go together")
    if slopes is not None:
        if not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32:
            raise TypeError("slopes must be a float32 torch.Tensor")
        if slopes.device != q.device:
            raise AssertionError("slopes must have the device of the first argument")
        if tuple(slopes.shape) != (nheads,):
            raise AssertionError(f"slopes must have shape {(nheads,)}, got {tuple(slopes.shape)}")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise AssertionError("slopes must not require gradients: none is formed")
        slopes = slopes.contiguous()
    if prefix is not None:
        prefix = _index(prefix, "prefix", q, (B,))
    if places is not None:
        places = _index(places, "places", q, tuple(q.shape[:2]))
    return _Shape(cap, slopes, prefix, places)


def _sliding(train, q, k, v, W, S, H, Hk, scale, lengths, shape=None):
    """y, and with train what the backward takes of the call."""
    (q, qr, qb), (k, kr, kb), (v, vr, vb) = _rows(q), _rows(k), _rows(v)
    B, n, C = q.shape
    y = torch.empty((B, n, C), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H * n), dtype=torch.float32, device=q.device) if train else None
    rest = torch.empty_like(y) if train and q.dtype != torch.float32 else None
    code = _CODES[q.dtype]
    rows = (q.data_ptr(), qr, qb, k.data_ptr(), kr, kb, v.data_ptr(), vr, vb, ptr(lengths), y.data_ptr(), ptr(rest), ptr(lse))
    if shape is None:
        _call(q.device, L.lib.circatt_sliding_fwd, code, n, B, H, Hk, C // H, W, S, scale, *rows)
    else:
        _call(q.device, L.lib.circatt_shaped_fwd, code, n, B, H, Hk, C // H, W, S, scale, *shape.args(), *rows)
    return y, (q, k, v, y, rest, lse, lengths), (code, W, S, H, Hk, scale, qr, qb, kr, kb, vr, vb)


class SlidingAttentionFn(torch.autograd.Function):
    """y of sliding_mh_attention (circatt_sliding_fwd / circatt_sliding_bwd)."""

    @staticmethod
    def forward(ctx, *args):
        y, saved, ctx.meta = _sliding(True, *args)
        ctx.save_for_backward(*saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return (*_sliding_gradients(ctx, dy, ctx.saved_tensors), None, None, None, None, None, None)


class ShapedAttentionFn(torch.autograd.Function):
    """The same with shaped scores (circatt_shaped_fwd / circatt_shaped_bwd).  The
    shape's arrays are arguments of their own, so that one that is written before
    the backward is noticed."""

    @staticmethod
    def forward(ctx, cap, slopes, prefix, places, *args):
        y, saved, ctx.meta = _sliding(True, *args, _Shape(cap, slopes, prefix, places))
        ctx.cap = cap
        ctx.save_for_backward(*saved, slopes, prefix, places)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        *saved, slopes, prefix, places = ctx.saved_tensors
        grads = _sliding_gradients(ctx, dy, saved, _Shape(ctx.cap, slopes, prefix, places), 4)
        return (None, None, None, None, *grads, None, None, None, None, None, None)


def _sliding_gradients(ctx, dy, saved, shape=None, first=0):
    """dq, dk, dv of a call; q is its Function's argument number `first`."""
    q, k, v, y, rest, lse, lengths = saved
    code, W, S, H, Hk, scale, qr, qb, kr, kb, vr, vb = ctx.meta
    B, n, C = q.shape
    dy, dr, db = _rows(dy)
    dq = torch.empty((B, n, C), dtype=q.dtype, device=q.device)
    dk = dv = None
    if ctx.needs_input_grad[first + 1] or ctx.needs_input_grad[first + 2]:
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dv = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    sizes = (code, n, B, H, Hk, C // H, W, S)
    if shape is None:
        wbytes = L.lib.circatt_sliding_bwd_workspace_bytes(*sizes)
    else:
        slopes, prefix, places = shape.arrays
        wbytes = L.lib.circatt_shaped_bwd_workspace_bytes(*sizes, slopes is not None,
                                                          1 if places is not None else 2 if prefix is not None else 0)
    work = torch.empty((max(wbytes, 4) // 4,), dtype=torch.float32, device=q.device)
    rows = (q.data_ptr(), qr, qb, k.data_ptr(), kr, kb, v.data_ptr(), vr, vb, ptr(lengths), y.data_ptr(), ptr(rest),
            lse.data_ptr(), dy.data_ptr(), dr, db, dq.data_ptr(), ptr(dk), ptr(dv), work.data_ptr(), wbytes)
    if shape is None:
        _call(q.device, L.lib.circatt_sliding_bwd, *sizes, scale, *rows)
    else:
        _call(q.device, L.lib.circatt_shaped_bwd, *sizes, scale, *shape.args(), *rows)
    return dq, dk, dv


def _window(W, sinks, scale, dh):
    W = _EVERY if W is None else int(W)
    if W < 1:
        raise AssertionError(f"window W={W} must be >= 1")
    if int(sinks) < 0:
        raise AssertionError(f"sinks={sinks} must be >= 0")
    # what holds every token; larger numbers would lose their high bits on the way to C
    return min(W, _EVERY), min(int(sinks), _EVERY), 1.0 / math.sqrt(dh) if scale is None else float(scale)


def sliding_mh_attention(q, k, v, W, nheads: int, *, kv_heads: int = None, sinks: int = 0, scale: float = None,
                         lengths: torch.Tensor = None, cap: float = None, slopes: torch.Tensor = None,
                         places: torch.Tensor = None, prefix: torch.Tensor = None) -> torch.Tensor:
    """Causal multi-head attention in a sliding window with sinks: token i of a
    signal sees the W tokens up to itself and the first ``sinks`` ones,

        y_i = sum_j softmax_j(scale <q_i, k_j>) v_j,  j <= i, j > i - W or j < sinks.

    q: (B, L, nheads*D); k, v: (B, L, kv_heads*D), each of their heads serving
    nheads/kv_heads heads of q (kv_heads None: as many as q's).  W None: every
    token up to i.  scale None: 1/sqrt(D).  lengths (int32, (B,)): a padded
    batch; rows from a signal's length on are zero, receive and give no
    gradient, and what they hold does not matter.  A row whose visible scores are
    all -inf is NaN.  Differentiable in q, k, v, once and not in forward mode.

    The scores x_ij = scale <q_i, k_j> may be shaped: into
    ``cap`` tanh(x_ij / cap) (with a scale above 0), and by - ``slopes``[h] |i - j| behind
    that (float32, (nheads,); not differentiable in them).  And what a token sees:
    places (int32, (B, L)): signals that hold documents one after another, each token's
    place in its own, 0, 1, 2, ... (as axial_rotary takes positions).  A token sees
    its own document alone, whose first tokens are its sinks.  Places that do not
    count up so give unspecified rows; those behind lengths are not looked at.
    prefix (int32, (B,)): every token of signal b sees the first prefix[b] ones too, those
    before them included.  Not together with places.
    Both are read on the device when the kernels run."""
    _require(q, "q")
    _require(k, "k", q)
    _require(v, "v", q)
    if q.dim() != 3 or k.dim() != 3:
        raise AssertionError("token signals are (B, L, C)")
    nheads = int(nheads)
    kv_heads = nheads if kv_heads is None else int(kv_heads)
    dh = _head_count(q.shape[2], nheads, "q's")
    if kv_heads < 1 or nheads % kv_heads != 0:
        raise AssertionError(f"nheads ({nheads}) must be divisible by kv_heads ({kv_heads})")
    if k.shape != v.shape or k.shape[:2] != q.shape[:2] or k.shape[2] != kv_heads * dh:
        raise AssertionError(f"k and v must be {(*q.shape[:2], kv_heads * dh)}, got {tuple(k.shape)} and "
                             f"{tuple(v.shape)}")
    W, sinks, scale = _window(W, sinks, scale, dh)
    if lengths is not None:
        lengths = _index(lengths, "lengths", q, (q.shape[0],))
    args = (q, k, v, W, sinks, nheads, kv_heads, scale, lengths)
    plain = not cap and slopes is None and prefix is None and places is None
    shape = None if plain else _shape(q, q.shape[0], nheads, cap, slopes, prefix, places)
    if _recorded(q, k, v):
        return SlidingAttentionFn.apply(*args) if shape is None else ShapedAttentionFn.apply(shape.cap, *shape.arrays, *args)
    return _sliding(False, *args, shape)[0]


def _cache(cache_k, cache_v, like):
    _require(cache_k, "cache_k", like)
    _require(cache_v, "cache_v", like)
    if cache_k.dim() != 3 or cache_k.shape != cache_v.shape:
        raise AssertionError("caches are (pages, page size, C), k's and v's alike")
    npages, page, C = cache_k.shape
    sp, sr, sc = cache_k.stride()
    if cache_k.stride() != cache_v.stride():
        raise AssertionError("the caches of k and v must have equal strides")
    if sc != 1 and C > 1:
        raise AssertionError("the channels of a cache's token must be adjacent")
    if page == 1:
        sr = C if npages == 1 else min(sp, 1 << 24)
    return npages, page, C, (sp if npages > 1 else page * sr), sr


def _table(pages, lengths, offsets, like):
    if not isinstance(pages, torch.Tensor) or pages.dtype != torch.int32 or pages.dim() != 2:
        raise TypeError("pages must be an int32 torch.Tensor (sequences, pages of each)")
    if pages.device != like.device:
        raise AssertionError("pages must have the type and the device of the first argument")
    if pages.stride(1) != 1 or pages.stride(0) < pages.shape[1]:
        pages = pages.contiguous()
    B = pages.shape[0]
    lengths = _index(lengths, "lengths", like, (B,))
    if offsets is not None:
        offsets = _index(offsets, "offsets", like, (B + 1,))
    return pages, B, lengths, offsets


def paged_mh_attention(q, cache_k, cache_v, pages, lengths, W, nheads: int, *, kv_heads: int = None, sinks: int = 0,
                       scale: float = None, offsets: torch.Tensor = None, out: torch.Tensor = None, cap: float = None,
                       slopes: torch.Tensor = None, prefix: torch.Tensor = None) -> torch.Tensor:
    """sliding_mh_attention of the new tokens of several sequences over a paged
    cache that holds their keys and values (paged_append_), without gradients.

    q: (T, nheads*D), the sequences' new tokens in order: sequence b has rows
    offsets[b] .. offsets[b+1] - 1 (int32, (B+1,); None: one row each, T = B).
    cache_k, cache_v: (pages, page size, kv_heads*D), the page size a power of
    two; token j of sequence b is row j % size of page pages[b, j // size]
    (int32, (B, most)); lengths (int32, (B,)) counts a sequence's tokens with
    the new ones.  The arrays of numbers are read on the device when the kernels
    run: a captured call follows what they hold then.  A page number that is not
    in the cache hides its tokens, and a token behind the table's last page sees
    nothing; a row that sees nothing is zero.  Offsets ascend from 0: others give
    unspecified rows.  Rows of q behind the last sequence give zero rows, or leave
    ``out``, which overlaps neither q nor the caches, alone where the caller
    passes it.  cap, slopes and prefix (one number for each sequence) as
    sliding_mh_attention takes them; of a prefix that is not yet in the cache the new
    tokens see what is."""
    _require(q, "q")
    if q.dim() != 2:
        raise AssertionError("q is (T, C): the new tokens of all sequences in order")
    npages, page, C, page_stride, row_stride = _cache(cache_k, cache_v, q)
    nheads = int(nheads)
    kv_heads = nheads if kv_heads is None else int(kv_heads)
    dh = _head_count(q.shape[1], nheads, "q's")
    if kv_heads < 1 or nheads % kv_heads != 0:
        raise AssertionError(f"nheads ({nheads}) must be divisible by kv_heads ({kv_heads})")
    if C != kv_heads * dh:
        raise AssertionError(f"the caches must hold {kv_heads * dh} channels a token, got {C}")
    W, sinks, scale = _window(W, sinks, scale, dh)
    pages, B, lengths, offsets = _table(pages, lengths, offsets, q)
    T = q.shape[0]
    q, q_row, _ = _rows(q.detach()[None])
    if out is None:
        y = torch.empty((T, nheads * dh), dtype=q.dtype, device=q.device)
    else:
        y = out
        _require(y, "out", q)
        if tuple(y.shape) != (T, nheads * dh) or not y.is_contiguous():
            raise AssertionError(f"out must be contiguous {(T, nheads * dh)}")
    shape = None if not cap and slopes is None and prefix is None else _shape(q, B, nheads, cap, slopes, prefix)
    code = _CODES[q.dtype]
    room = (code, T, B, nheads, kv_heads, dh, W, sinks, page, pages.shape[1])
    wbytes = (L.lib.circatt_paged_workspace_bytes(*room) if prefix is None
              else L.lib.circatt_shaped_paged_workspace_bytes(*room, 1))
    work = torch.empty((wbytes // 4,), dtype=torch.float32, device=q.device) if wbytes > 0 else None
    sizes = (code, T, B, nheads, kv_heads, dh, W, sinks, scale)
    rest = (q.data_ptr(), q_row, cache_k.data_ptr(), cache_v.data_ptr(), npages, page, page_stride, row_stride,
            pages.data_ptr(), pages.stride(0), pages.shape[1], lengths.data_ptr(), ptr(offsets), y.data_ptr(),
            1 if out is None else 0, ptr(work), wbytes)
    if shape is None:
        _call(q.device, L.lib.circatt_paged_attention, *sizes, *rest)
    else:
        _call(q.device, L.lib.circatt_shaped_paged, *sizes, *shape.args()[:3], *rest)
    if out is not None:
        increment_version(out)
    return y


def paged_append_(cache_k, cache_v, k, v, pages, lengths, *, offsets: torch.Tensor = None) -> None:
    """Writes the new tokens' keys and values, k and v (T, C), into the caches
    (pages, page size, C): the arguments of paged_mh_attention, lengths counting
    the new tokens.  A token whose page number is not in the cache is dropped;
    no two tokens may share a slot, and k and v hold no slot that is written."""
    _require(k, "k")
    _require(v, "v", k)
    npages, page, C, page_stride, row_stride = _cache(cache_k, cache_v, k)
    if k.dim() != 2 or k.shape != v.shape or k.shape[1] != C:
        raise AssertionError(f"k and v must be (T, {C}), got {tuple(k.shape)} and {tuple(v.shape)}")
    pages, B, lengths, offsets = _table(pages, lengths, offsets, k)
    k, v = (t.detach() if t.stride(1) == 1 or C == 1 else t.detach().contiguous() for t in (k, v))
    _call(k.device, L.lib.circatt_paged_append, _CODES[k.dtype], k.shape[0], B, C, k.data_ptr(), k.stride(0), v.data_ptr(),
          v.stride(0), cache_k.data_ptr(), cache_v.data_ptr(), npages, page, page_stride, row_stride, pages.data_ptr(),
          pages.stride(0), pages.shape[1], lengths.data_ptr(), ptr(offsets))
    increment_version((cache_k, cache_v))


def _held(pages, lengths, counts, like):
    """The table, lengths and counts of a cache's pages, checked."""
    if not isinstance(pages, torch.Tensor) or pages.dtype != torch.int32 or pages.dim() != 2:
        raise TypeError("pages must be an int32 torch.Tensor (sequences, pages of each)")
    if not pages.is_cuda:
        raise ValueError("pages must live on a HIP device (libcircatt has no CPU path)")
    if like is not None and pages.device != like.device:
        raise AssertionError("pages must have the device of the cache")
    if pages.shape[0] < 1 or pages.shape[1] < 1:
        raise AssertionError(f"a page table of {tuple(pages.shape)}")
    if pages.stride(1) != 1 and pages.shape[1] > 1 or pages.stride(0) < pages.shape[1]:
        pages = pages.contiguous()
    if lengths is not None:
        lengths = _index(lengths, "lengths", pages, (pages.shape[0],))
    if not isinstance(counts, torch.Tensor) or counts.dim() != 1:
        raise TypeError("counts must be an int32 torch.Tensor (pages of the cache,)")
    counts = _index(counts, "counts", pages, tuple(counts.shape) if like is None else (like.shape[0],))
    return pages, max(pages.stride(0), pages.shape[1]), lengths, counts


def paged_fork(pages, lengths, counts, source, page_size: int):
    """The tables of sequences that go on from others: (pages, lengths, counts) with row n
    as sequence source[n] had it (int32, (N,); a number outside the old sequences
    gives an empty one).  The sequences share their pages; no token moves.

    pages (int32, (B, most)) and lengths (int32, (B,)) as paged_mh_attention takes
    them; counts (int32, (pages of the cache,)) says how often each page is held, 0 for a
    free one.  Old sequences that nobody goes on from give their pages back.
    Page numbers outside the cache are kept and not counted."""
    pages, row, lengths, counts = _held(pages, lengths, counts, None)
    if not isinstance(source, torch.Tensor) or source.dim() != 1:
        raise TypeError("source must be an int32 torch.Tensor (sequences,)")
    source = _index(source, "source", pages, tuple(source.shape))
    (B, most), N = pages.shape, source.shape[0]
    new = pages.new_empty((N, most)), torch.empty_like(source), torch.empty_like(counts)
    _call(pages.device, L.lib.circatt_paged_fork, B, counts.shape[0], int(page_size), pages.data_ptr(), row, most,
          lengths.data_ptr(), counts.data_ptr(), N, ptr(source), ptr(new[0]), ptr(new[1]), new[2].data_ptr())
    return new


def paged_resize_(cache_k, cache_v, pages, lengths, counts, to):
    """The tables of sequences that grow, shrink or end: (pages, lengths, counts) with
    sequence b at to[b] tokens (int32, (B,); no more than its row of the table holds;
    below 0: as it is), so that paged_append_ finds pages for the new ones.

    Pages behind the new lengths are given back.  Then sequences get what they lack, in
    their order, the free pages of the lowest numbers first.  A sequence that grows
    from within a page that is held more than once gets its own copy of that page's
    tokens, the only ones that move; of several that do so in one call each gets one.  One that
    shrinks gets none: a step that takes tokens off a sequence and brings it new ones
    resizes it twice, to what stays of it and then to that with the new ones (an append
    behind one resize to fewer tokens may write into a page that others hold).  From the first sequence on that finds too few free
    pages, those that need any stay as they are, as the lengths that come back show.
    Other arguments as paged_fork's."""
    npages, page, C, page_stride, row_stride = _cache(cache_k, cache_v, cache_k)
    pages, row, lengths, counts = _held(pages, lengths, counts, cache_k)
    B, most = pages.shape
    to = _index(to, "to", pages, (B,))
    new = pages.new_empty((B, most)), torch.empty_like(lengths), torch.empty_like(counts)
    wbytes = L.lib.circatt_paged_resize_workspace_bytes(B, npages)
    work = pages.new_empty(max(wbytes, 4) // 4)
    _call(pages.device, L.lib.circatt_paged_resize, _CODES[cache_k.dtype], C, cache_k.data_ptr(), cache_v.data_ptr(), npages,
          page, page_stride, row_stride, B, pages.data_ptr(), row, most, lengths.data_ptr(), counts.data_ptr(), to.data_ptr(),
          *(t.data_ptr() for t in new), work.data_ptr(), wbytes)
    increment_version((cache_k, cache_v))
    return new


def paged_compact_(cache_k, cache_v, pages, counts):
    """The tables of a cache whose held pages have moved to its lowest numbers, with
    their tokens: (pages, counts).  The held pages from number ``used`` on, as many as
    there are held ones, take the free numbers below it in order.  Every table that
    refers to the cache is one: its rows may be those of several, joined.  Other
    arguments as paged_fork's."""
    npages, page, C, page_stride, row_stride = _cache(cache_k, cache_v, cache_k)
    pages, row, _, counts = _held(pages, None, counts, cache_k)
    B, most = pages.shape
    new = pages.new_empty((B, most)), torch.empty_like(counts)
    wbytes = L.lib.circatt_paged_compact_workspace_bytes(npages)
    work = pages.new_empty(max(wbytes, 4) // 4)
    _call(pages.device, L.lib.circatt_paged_compact, _CODES[cache_k.dtype], C, cache_k.data_ptr(), cache_v.data_ptr(), npages,
          page, page_stride, row_stride, B, pages.data_ptr(), row, most, counts.data_ptr(), *(t.data_ptr() for t in new),
          work.data_ptr(), wbytes)
    increment_version((cache_k, cache_v))
    return new


def _token_stride(x):
    """(x, elements from token to token): one distance over all leading dims."""
    C = x.shape[-1]
    if x.is_contiguous():
        return x, C
    row = None
    if x.stride(-1) == 1 or C == 1:
        step = None
        for n, s in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
            if n == 1:
                continue
            if step is None:
                row = step = s
            elif s != step:
                row = -1
                break
            step = step * n
        if row is None:
            row = C
    if row is None or row < C:
        return x.contiguous(), C
    return x, row


class AxialRotaryFn(torch.autograd.Function):
    """The turn of axial_rotary (circatt_axial_rotary); its pullback is the turn
    the other way."""

    @staticmethod
    def forward(ctx, x, positions, *meta):
        ctx.meta = meta
        ctx.save_for_backward(positions)
        return _turn(x, 0, *meta, positions)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (positions,) = ctx.saved_tensors
        return _turn(g, 1, *ctx.meta, positions), None, None, None, None, None, None, None


def _turn(x, inverse, grid, pairs, H, base, per_image, interleaved, positions):
    x, row = _token_stride(x)
    shape = x.shape
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    C = shape[-1]
    nb, P = (shape[0], math.prod(shape[1:-1])) if len(shape) > 2 else (1, shape[0])
    n1, n2, n3 = grid
    p1, p2, p3 = (*pairs, 0, 0)[:3]
    _call(x.device, L.lib.circatt_axial_rotary_wide, _CODES[x.dtype], inverse, 1 if interleaved else 0, len(pairs), n1, n2,
          n3, P, nb, H, C // H, p1, p2, p3, *base, x.data_ptr(), row, ptr(positions),
          P * len(pairs) if per_image else 0, y.data_ptr())
    return y


def axial_rotary(x, pairs, nheads: int, *, base: float = 10000.0, positions: torch.Tensor = None,
                 interleaved: bool = False) -> torch.Tensor:
    """Rotary positions on one to three axes, for queries and keys of attention
    on lines, images (also the fused circulant attention's, channels-last) and
    video: pairs = (p1, ...) pairs of every head turn with each axis, pair i of
    an axis by position * base^(-i/p).  A head's first 2*p1 channels belong to
    axis 1, the next 2*p2 to axis 2, and so on; the channels behind stay.  Pair i
    is channels i and i + p of its section, or 2i and 2i + 1 when interleaved.

    x: (B, *reversed(spatial), C) with nheads heads in C, or packed tokens
    (T, C).  positions None: the grid's own, axis 1 the fastest spatial axis, as
    many axes as spatial ones.  Else int32, (*x.shape[:-1], axes), or without
    the batch dim to share them.  The angle is formed in 64 bits, from the base as
    it is given.  Float32, Float16, BFloat16; differentiable in x, once and not in
    forward mode."""
    _require(x, "x")
    if x.dim() < 2:
        raise AssertionError("x is (B, *spatial, C) or (T, C)")
    pairs = tuple(min(max(int(p), 0), _EVERY) for p in pairs)  # (refused by C as they are)
    if not 1 <= len(pairs) <= 3:
        raise AssertionError(f"{len(pairs)} axes; 1 to 3 are supported")
    _head_count(x.shape[-1], int(nheads), "x's")
    grid, per_image = (1, 1, 1), False
    if positions is None:
        spatial = tuple(reversed(x.shape[1:-1]))
        if len(spatial) != len(pairs):
            raise AssertionError(f"{len(pairs)} axes for {len(spatial)} spatial dims: give positions")
        grid = (*spatial, 1, 1)[:3]
    else:
        if not isinstance(positions, torch.Tensor):
            raise TypeError("positions must be an int32 torch.Tensor")
        per_image = x.dim() > 2 and positions.dim() == x.dim()
        shape = x.shape[:-1] if per_image or x.dim() == 2 else x.shape[1:-1]
        positions = _index(positions, "positions", x, (*shape, len(pairs)))
    base = float(base)
    near = ctypes.c_float(base).value
    meta = (grid, pairs, int(nheads), (near, base - near), per_image, bool(interleaved))
    if _recorded(x):
        return AxialRotaryFn.apply(x, positions, *meta)
    return _turn(x, 0, *meta, positions)


__all__ = ["axial_rotary", "paged_append_", "paged_compact_", "paged_fork", "paged_mh_attention", "paged_resize_",
           "sliding_mh_attention"]
