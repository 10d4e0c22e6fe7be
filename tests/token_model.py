"""64-bit restatement of the token operators, with element-wise bounds of the
error that the kernels' arithmetic allows.

Bounds count half steps u of the element type (and 2^-24 of Float32 sums):
  e    relative error of a probability: Float32 scores of D products are off by
       (D + 3) 2^-24 scale <|q|, |k|>, twice that with the maximum's, and exp2,
       the sum of n terms and the division add (n + 16) 2^-24
  y    (u + e) P|V| for the rounded probabilities, u |y| for the output
  dV   the same with P'|dO|
  D    = rowsum(dO y) of the rounded y: (u|y| + bound of y) . |dO|
  dS   = P (dP - D): (u + e) |dS| + P (bound of D + (D + 3) 2^-24 |dO|.|V|)
  dQ, dK  scale times the bound of dS against |K|, |Q|, and u of the result
Elements too small for Float16's normal range are off by 2^-25 each instead."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def visible(pos, n, W, S):
    """(rows, n): row at position pos[r] sees key j."""
    j = torch.arange(n)
    return (j[None] <= pos[:, None]) & ((j[None] > pos[:, None] - W) | (j[None] < S))


def attention(q, k, v, see, scale, dtype, dy=None):
    """One head in 64 bits: q (r, D), k, v (n, D), see (r, n).  Returns
    [(value, bound), ...] for y, or y, dq, dk, dv with dy.  Rows of k and v that
    no row sees take no part, whatever they hold."""
    u, tiny = HALF[dtype], TINY[dtype]
    f = 2.0 ** -24
    n, D = k.shape
    used = see.any(0)
    k = torch.where(used[:, None], k, torch.zeros_like(k))
    v = torch.where(used[:, None], v, torch.zeros_like(v))
    s = torch.where(see, (q @ k.T) * scale, torch.full((), -math.inf, dtype=torch.float64))
    m = s.amax(1, keepdim=True)
    p = torch.where(see, torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m))), torch.zeros_like(s))
    p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    absqk = torch.where(see, (q.abs() @ k.abs().T) * scale, torch.zeros_like(s))
    e = 2 * (D + 3) * f * absqk.amax(1, keepdim=True) + (n + 16) * f
    y = p @ v
    pv = p @ v.abs()
    by = (u + e) * pv + u * y.abs() + tiny * (v.abs().sum(0) + 1) + 1e-30
    if dy is None:
        return [(y, by)]
    dv = p.T @ dy
    bdv = p.T @ ((u + e) * dy.abs()) + u * dv.abs() + tiny * (dy.abs().sum(0) + 1) + 1e-30
    d = (dy * y).sum(1, keepdim=True)
    bd = ((u * y.abs() + by) * dy.abs()).sum(1, keepdim=True) + D * f * (dy * y).abs().sum(1, keepdim=True)
    dp = dy @ v.T
    ds = p * (dp - d)
    bds = (u + e) * ds.abs() + p * (bd + (D + 3) * f * (dy.abs() @ v.abs().T)) + tiny
    bds = torch.where(see, bds, torch.zeros_like(bds))
    dq, dk = scale * (ds @ k), scale * (ds.T @ q)
    n_r = q.shape[0]
    bdq = scale * (bds @ k.abs()) + (u + n * f) * scale * (ds.abs() @ k.abs()) + tiny + 1e-30
    bdk = scale * (bds.T @ q.abs()) + (u + n_r * f) * scale * (ds.abs().T @ q.abs()) + tiny + 1e-30
    return [(y, by), (dq, bdq), (dk, bdk), (dv, bdv)]


def sliding(q, k, v, W, H, Hk, S, scale, lengths, dtype, dy=None):
    """The whole operator on (B, L, C) tensors in 64 bits: [(value, bound), ...].
    A shared head's bounds add up, and its sum is rounded once: covered by the
    sums of the single heads' bounds."""
    B, L, C = q.shape
    D = C // H
    out = [[torch.zeros_like(t) for _ in range(2)] for t in ((q,) if dy is None else (q, q, k, v))]
    for b in range(B):
        n = L if lengths is None else max(0, min(L, int(lengths[b])))
        see = visible(torch.arange(n), n, W, S)
        for h in range(H if n else 0):
            hq, g = slice(h * D, h * D + D), h // (H // Hk)
            hk = slice(g * D, g * D + D)
            got = attention(q[b, :n, hq], k[b, :n, hk], v[b, :n, hk], see, scale, dtype,
                            None if dy is None else dy[b, :n, hq])
            for (val, bound), (x, bx), cols in zip(out, got, (hq, hq, hk, hk)):
                val[b, :n, cols] += x
                bound[b, :n, cols] += bx
    return out


def paged(q, cache_k, cache_v, pages, lengths, offsets, W, H, Hk, S, scale, dtype):
    """(value, bound) of (T, C) in 64 bits; rows behind the last sequence zero."""
    T, C = q.shape
    D, page = C // H, cache_k.shape[1]
    y, by = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(len(lengths)):
        lo, hi = int(offsets[b]), int(offsets[b + 1])
        n = max(0, int(lengths[b]))
        if hi <= lo:
            continue
        pos = torch.arange(n - (hi - lo), n)
        held = min(n, pages.shape[1] * page)
        j = torch.arange(held)
        pg = pages[b].long()[j // page] if held else torch.zeros(0, dtype=torch.long)
        there = (pg >= 0) & (pg < cache_k.shape[0])
        slot = torch.where(there, pg, torch.zeros_like(pg))
        kk, vv = cache_k[slot, j % page], cache_v[slot, j % page]
        see = visible(pos, held, W, S) & there[None] & (pos < pages.shape[1] * page)[:, None]
        for h in range(H):
            hq, g = slice(h * D, h * D + D), h // (H // Hk)
            hk = slice(g * D, g * D + D)
            if held == 0:
                continue
            ((x, bx),) = attention(q[lo:hi, hq], kk[:, hk], vv[:, hk], see, scale, dtype)
            y[lo:hi, hq], by[lo:hi, hq] = x, bx
    return y, by


def rotary(x, pairs, H, base, positions, interleaved, dtype, inverse=False):
    """(value, bound): x (..., C) in 64 bits, positions (..., axes) integers.
    Cosine and sine are off by 2^-21 at most: 2^-24 of a turn in the reduced
    angle and the hardware's 1.2e-7."""
    D = x.shape[-1] // H
    h = x.reshape(*x.shape[:-1], H, D)
    out, size = h.clone(), h.abs().clone() * 0
    at = 0
    for a, p in enumerate(pairs):
        f = base ** (-torch.arange(p, dtype=torch.float64) / p)
        ang = positions[..., a].double()[..., None, None] * f
        c, s = torch.cos(ang), torch.sin(ang)
        if inverse:
            s = -s
        i = torch.arange(p) * 2 + at if interleaved else torch.arange(p) + at
        j = i + 1 if interleaved else i + p
        u, w = h[..., i], h[..., j]
        out[..., i], out[..., j] = u * c - w * s, u * s + w * c
        size[..., i] = size[..., j] = u.abs() + w.abs()
        at += 2 * p
    out, size = out.reshape(x.shape), size.reshape(x.shape)
    return out, HALF[dtype] * out.abs() + (2.0 ** -21 + 2.0 ** -23) * size + TINY[dtype]


def check(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    if bad.any():
        i = tuple(int(t[0]) for t in torch.nonzero(bad, as_tuple=True))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} elements off, the first at {i}: "
                             f"{got[i].item()} for {want[i].item()}, bound {bound[i].item()}")
