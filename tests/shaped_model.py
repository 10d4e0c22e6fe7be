"""64-bit restatement of the token attention with shaped scores, with element-wise
bounds of the error that the kernels' arithmetic allows, in the manner of
token_model.py (half steps u of the element type, f = 2^-24 of Float32).

The score s = cap tanh(x / cap) - slope |i - j|, x = scale <q, k>:
  x     D products and sums: (D + 3) f scale <|q|, |k|>, and as much of s at most
  tanh  the kernels form r = 1 / (1 + E), E = 2^(u x), and 1 - 2 r.  E's relative error
        is 2^-23 (exponential) and 2 f ln 2 of its exponent z (two roundings); with
        r (1 - r) <= 1/4 and z r (1 - r) <= 0.23 the tangent is off by 2^-24 + 2^-23 * 0.32 from it, by
        3 * 2^-23 from the reciprocal and the sum in it, and by f in the end: 2^-21 at
        most in all.  Where the series is taken instead, 8 f of the tangent: the fine
        form is off by max(8 f, 2^-21 / 0.33) <= 2^-19 of its value.
  bias  three roundings, and one of every partial sum: 4 f (|s| + cap + bias)
A probability p_j = exp(s_j - lse) is off by the error of its own score, the mean of
its row's (the sum), and (n + 16) f as in token_model.py, and where it is formed from
the stored lse by 2 f |lse| more.  The derivative 1 - t^2 is off by twice the
tangent's error and 4 f."""
import math

import torch

from token_model import HALF, TINY, check  # noqa: F401  (check: for the tests)

F = 2.0 ** -24


def attention(q, k, v, see, scale, dtype, cap=0.0, bias=None, dy=None):
    """One head in 64 bits: q (r, D), k, v (n, D), see (r, n), bias (r, n) or None (what
    is taken off the scores).  [(value, bound), ...] for y, or y, dq, dk, dv."""
    u, tiny = HALF[dtype], TINY[dtype]
    n, D = k.shape
    used = see.any(0)
    k = torch.where(used[:, None], k, torch.zeros_like(k))
    v = torch.where(used[:, None], v, torch.zeros_like(v))
    x = (q @ k.T) * scale
    es = (D + 3) * F * (q.abs() @ k.abs().T) * scale
    fine = dtype == torch.float32 or cap > 256
    bend, ebend = torch.ones_like(x), torch.zeros_like(x)
    s = x
    if cap:
        t = torch.tanh(x / cap)
        s = cap * t
        et = 2.0 ** -19 * t.abs() if fine else torch.full_like(t, 2.0 ** -21)
        bend, ebend = 1 - t * t, 2 * t.abs() * (et + es / cap * (1 - t * t)) + et * et + 4 * F
        es = torch.minimum(es, es * 0 + 2 * cap) + cap * et
    if bias is not None:
        s = s - bias
        es = es + 4 * F * (s.abs() + cap + bias)
    es = es + 2 * F * s.abs()
    zero = torch.zeros_like(s)
    s = torch.where(see, s, torch.full((), -math.inf, dtype=torch.float64))
    m = s.amax(1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    p = torch.where(see, torch.exp(s - m), zero)
    total = p.sum(1, keepdim=True).clamp(min=1e-300)
    p = p / total
    lse = (m + torch.log(total)).abs() * 2 * F
    es = torch.where(see, es, zero)
    e = es + (p * es).sum(1, keepdim=True) + (n + 16) * F
    y = p @ v
    by = (p * (u + e)) @ v.abs() + u * y.abs() + tiny * (v.abs().sum(0) + 1) + 1e-30
    if dy is None:
        return [(y, by)]
    e = e + lse
    dv = p.T @ dy
    bdv = (p * (u + e)).T @ dy.abs() + u * dv.abs() + tiny * (dy.abs().sum(0) + 1) + 1e-30
    d = (dy * y).sum(1, keepdim=True)
    bd = ((u * y.abs() + by) * dy.abs()).sum(1, keepdim=True) + D * F * (dy * y).abs().sum(1, keepdim=True)
    ds = p * (dy @ v.T - d)
    bds = e * ds.abs() + p * (bd + (D + 3) * F * (dy.abs() @ v.abs().T))
    dx = ds * bend
    bdx = torch.where(see, u * dx.abs() + bds * (bend + ebend) + ds.abs() * ebend + tiny, zero)
    n_r = q.shape[0]
    dq, dk = scale * (dx @ k), scale * (dx.T @ q)
    bdq = scale * (bdx @ k.abs()) + (u + n * F) * scale * (dx.abs() @ k.abs()) + tiny + 1e-30
    bdk = scale * (bdx.T @ q.abs()) + (u + n_r * F) * scale * (dx.abs().T @ q.abs()) + tiny + 1e-30
    return [(y, by), (dq, bdq), (dk, bdk), (dv, bdv)]


def visible(pos, n, W, S, start=None, P=0):
    """(rows, n): the row at position pos[r], whose document begins at start[r], sees
    key j."""
    j = torch.arange(n)[None]
    i = pos[:, None]
    first = torch.zeros_like(i) if start is None else start[:, None]
    return ((j >= first) & (j <= i) & ((j > i - W) | (j < first + S))) | ((j < P) & (i >= 0))


def sliding(q, k, v, W, H, Hk, S, scale, lengths, dtype, cap=0.0, slopes=None, places=None, prefix=None, dy=None):
    """The whole operator on (B, L, C) tensors in 64 bits: [(value, bound), ...]."""
    B, L, C = q.shape
    D = C // H
    out = [[torch.zeros_like(t) for _ in range(2)] for t in ((q,) if dy is None else (q, q, k, v))]
    for b in range(B):
        n = L if lengths is None else max(0, min(L, int(lengths[b])))
        if n == 0:
            continue
        i = torch.arange(n)
        start = None if places is None else (i - places[b, :n].long())
        see = visible(i, n, W, S, start, 0 if prefix is None else max(0, min(n, int(prefix[b]))))
        back = (i[:, None] - i[None]).abs().double()
        for h in range(H):
            hq, g = slice(h * D, h * D + D), h // (H // Hk)
            hk = slice(g * D, g * D + D)
            got = attention(q[b, :n, hq], k[b, :n, hk], v[b, :n, hk], see, scale, dtype, cap or 0.0,
                            None if slopes is None else back * float(slopes[h]), None if dy is None else dy[b, :n, hq])
            for (val, bound), (x, bx), cols in zip(out, got, (hq, hq, hk, hk)):
                val[b, :n, cols] += x
                bound[b, :n, cols] += bx
    return out


def paged(q, cache_k, cache_v, pages, lengths, offsets, W, H, Hk, S, scale, dtype, cap=0.0, slopes=None, prefix=None):
    """(value, bound) of (T, C) in 64 bits; rows behind the last sequence zero."""
    T, C = q.shape
    D, page = C // H, cache_k.shape[1]
    y, by = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(len(lengths)):
        lo, hi = int(offsets[b]), int(offsets[b + 1])
        n = max(0, int(lengths[b]))
        held = min(n, pages.shape[1] * page)
        if hi <= lo or held == 0:
            continue
        pos = torch.arange(n - (hi - lo), n)
        pos = torch.where(pos < pages.shape[1] * page, pos, torch.full_like(pos, -1))
        j = torch.arange(held)
        pg = pages[b].long()[j // page]
        there = (pg >= 0) & (pg < cache_k.shape[0])
        slot = torch.where(there, pg, torch.zeros_like(pg))
        kk, vv = cache_k[slot, j % page], cache_v[slot, j % page]
        P = 0 if prefix is None else max(0, min(held, int(prefix[b])))
        see = visible(pos, held, W, S, None, P) & there[None] & (pos >= 0)[:, None]
        back = (pos[:, None] - j[None]).abs().double()
        for h in range(H):
            hq, g = slice(h * D, h * D + D), h // (H // Hk)
            hk = slice(g * D, g * D + D)
            ((x, bx),) = attention(q[lo:hi, hq], kk[:, hk], vv[:, hk], see, scale, dtype, cap or 0.0,
                                   None if slopes is None else back * float(slopes[h]))
            y[lo:hi, hq], by[lo:hi, hq] = x, bx
    return y, by
