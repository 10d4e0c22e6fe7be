"""Performance cases of the token operators: causal sliding-window attention
with sinks (forward and training), the same attention over a paged cache, the
cache's append, and rotary positions with several axes.

A case is a dict of plain values; "op" says which operator:

  "sliding"  y = sliding_mh_attention(q, k, v, W, heads, ...) on (batch, length,
             channels) signals; train: the gradients of q, k, v as well;
             ragged: a padded batch with a length for each signal
  "paged"    y = paged_mh_attention(q, cache_k, cache_v, pages, lengths, ...):
             the new tokens of every sequence over a paged cache; new = 1: one
             token for each sequence; mixed: some sequences bring one token
  "append"   paged_append_(cache_k, cache_v, k, v, pages, lengths, ...)
  "rotary"   y = axial_rotary(x, pairs, heads, ...); train: the gradient too;
             given: positions are a tensor of the caller, else the grid's own

"spread" seeds the lengths of the sequences, which belong to the case; inputs
and the order of the pages come from the seed of prepare().
"""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "circulantattention.jl_amd")
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ca():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import circulant_attention
    return circulant_attention


def _sliding(name, batch, length, heads, kv_heads, dim, window, sinks, dtype, *, train=False, ragged=False, spread=0):
    return {"name": name, "op": "sliding", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "window": window, "sinks": sinks, "dtype": dtype, "train": train, "ragged": ragged,
            "spread": spread}


def _paged(name, batch, context, new, heads, kv_heads, dim, window, sinks, page, dtype, *, mixed=False, pad=0, spread=0):
    return {"name": name, "op": "paged", "batch": batch, "context": context, "new": new, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "page": page, "dtype": dtype,
            "mixed": mixed, "pad": pad, "spread": spread}


def _append(name, batch, context, new, kv_heads, dim, page, dtype, *, mixed=False, pad=0, spread=0):
    return {"name": name, "op": "append", "batch": batch, "context": context, "new": new, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "mixed": mixed, "pad": pad, "spread": spread}


def _rotary(name, batch, n1, n2, n3, heads, dim, p1, p2, p3, dtype, *, train=False, given=False, interleaved=False):
    return {"name": name, "op": "rotary", "batch": batch, "n1": n1, "n2": n2, "n3": n3, "heads": heads, "dim": dim,
            "p1": p1, "p2": p2, "p3": p3, "dtype": dtype, "train": train, "given": given, "interleaved": interleaved}


def listed():
    return [
        # a short signal of a small Float32 model: latency and launches
        _sliding("sliding_small", 1, 96, 4, 4, 32, 32, 4, "f32"),
        # a long prompt, eight heads of keys, no gradients
        _sliding("sliding_prompt", 1, 8192, 32, 8, 128, 1024, 4, "bf16"),
        # a training step on full sequences
        _sliding("sliding_train", 2, 4096, 16, 4, 128, 512, 4, "bf16", train=True),
        # a padded training batch of odd lengths, heads of 80, many sinks
        _sliding("sliding_train_ragged", 3, 1531, 12, 4, 80, 257, 17, "f16", train=True, ragged=True, spread=5),
        # one user's next token
        _paged("token_one_user", 1, 700, 1, 8, 2, 64, 4096, 4, 16, "bf16"),
        # the next token of a full serving batch, long contexts
        _paged("token_batch", 64, 8192, 1, 32, 8, 128, 4096, 4, 16, "bf16", spread=7),
        # chunks of two long prompts
        _paged("chunk_prompt", 2, 12000, 512, 32, 8, 128, 4096, 4, 64, "bf16", spread=3),
        # a serving batch that mixes single tokens with chunks; plain causal
        # attention (the window holds everything), odd group of heads
        _paged("chunk_mixed", 33, 2500, 128, 15, 5, 96, 1 << 20, 0, 32, "f16", mixed=True, pad=11, spread=9),
        # the new keys and values of a serving batch's tokens, and of chunks
        _append("append_token_batch", 64, 1024, 1, 8, 128, 16, "bf16", spread=7),
        _append("append_chunks", 4, 6000, 4096, 8, 128, 64, "bf16", pad=5, spread=3),
        # feature maps of 64 channels in four heads, as the attention on images
        # takes them, with the gradient
        _rotary("rotary_image_train", 4, 256, 256, 0, 4, 16, 4, 4, 0, "f32", train=True),
        # video tokens, positions given
        _rotary("rotary_video", 1, 80, 45, 16, 16, 128, 22, 21, 16, "bf16", given=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# the most that a drawn case takes, by operator: the scores of the plain form
# (rows x keys x heads), or the values moved
_MOST = {"sliding": 32 * 8192 ** 2, "sliding_train": 2 * 16 * 4096 ** 2, "paged": 64 * 32 * 8192,
         "chunk": 2 * 32 * 512 * 12000, "append": 4 * 4096 * 1024 * 2, "rotary": 4 * 256 * 256 * 64 * 2}


def draw(rng):
    """Signals of 1 to 8192 tokens, contexts of 1 to 16384, chunks of 1 to 4096,
    windows of 1 to everything, heads of 8 to 128 channels in groups of 1 to 8,
    grids of one to three axes; all three types."""
    dtype = rng.choice(["bf16"] * 5 + ["f16"] * 3 + ["f32"] * 2)
    dim = rng.choice([8, 16, 32, 40, 64, 64, 72, 80, 96, 104, 128, 128, 128])
    kv_heads, group = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    window = rng.choice([_log_int(rng, 1, 8192), _log_int(rng, 32, 4096), 1 << 20])
    sinks = rng.choice([0, 0, 1, 4, 4, rng.randint(2, 64), rng.randint(65, 700)])
    spread = rng.randint(0, 1 << 20)
    op = rng.choice(["sliding"] * 5 + ["paged"] * 5 + ["append"] * 2 + ["rotary"] * 3)
    while True:
        if op == "sliding":
            train = rng.random() < 0.6
            c = _sliding("", rng.choice([1, 1, 2, 3, 5, 8]), _log_int(rng, 1, 8192), kv_heads * group, kv_heads, dim,
                         window, sinks, dtype, train=train, ragged=rng.random() < 0.4, spread=spread)
            cost, most = c["batch"] * c["heads"] * c["length"] ** 2, _MOST["sliding_train" if train else "sliding"]
        elif op == "paged":
            one = rng.random() < 0.5
            context = _log_int(rng, 1, 16384)
            new = 1 if one else min(context, _log_int(rng, 1, 1024))
            c = _paged("", _log_int(rng, 1, 128 if one else 40), context, new, kv_heads * group, kv_heads, dim, window,
                       sinks, rng.choice([8, 16, 16, 32, 64, 128]), dtype, mixed=not one and rng.random() < 0.5,
                       pad=0 if one else rng.choice([0, 0, 1, 9]), spread=spread)
            cost = c["batch"] * c["heads"] * new * context
            # the plain form reads its caches in 32 bits; one token a sequence is bound by that
            cost, most = (cost * dim // 128, _MOST["paged"]) if one else (cost, _MOST["chunk"])
            if c["batch"] * context * kv_heads * dim > 64 * 8192 * 1024:
                continue
        elif op == "append":
            context = _log_int(rng, 1, 8192)
            c = _append("", _log_int(rng, 1, 64), context, min(context, rng.choice([1, _log_int(rng, 1, 4096)])),
                        kv_heads, dim, rng.choice([8, 16, 16, 32, 64, 128]), dtype, mixed=rng.random() < 0.3,
                        pad=rng.choice([0, 0, 3]), spread=spread)
            cost, most = c["batch"] * context * kv_heads * dim * 2, _MOST["append"] * 2
        else:
            axes = rng.choice([1, 2, 2, 3, 3])
            half = dim // 2
            cut = sorted(rng.randint(1, half) for _ in range(axes - 1)) if axes > 1 else []
            p = [b - a for a, b in zip([0] + cut, cut + [half - rng.choice([0, 0, half // 4])])]
            if min(p) < 1:
                continue
            n = [_log_int(rng, 1, (65536, 512, 64)[axes - 1]) for _ in range(axes)]
            p, n = p + [0] * (3 - axes), n + [0] * (3 - axes)
            c = _rotary("", rng.choice([1, 2, 3, 4]), n[0], n[1], n[2], kv_heads * group, dim, p[0], p[1], p[2], dtype,
                        train=rng.random() < 0.4, given=rng.random() < 0.5, interleaved=rng.random() < 0.3)
            cost = c["batch"] * math.prod(max(1, x) for x in n) * c["heads"] * dim * (2 if c["train"] else 1)
            most = _MOST["rotary"]
        if cost <= most:
            del c["name"]
            return c
        kv_heads, group = rng.choice([1, 2, 3, 4]), rng.choice([1, 2, 3, 4])


# ---------------------------------------------------------------------------
# sizes that belong to the case
# ---------------------------------------------------------------------------
def _signal_lengths(c):
    """The padded batch's lengths: the longest fills the signal."""
    if not c["ragged"]:
        return [c["length"]] * c["batch"]
    r = random.Random(c["spread"])
    return [c["length"]] + [r.randint(c["length"] // 3, c["length"]) for _ in range(c["batch"] - 1)]


def _sequences(c):
    """(tokens in the cache, new ones among them) for each sequence."""
    r = random.Random(c["spread"])
    out = []
    for b in range(c["batch"]):
        n = c["context"] if b == 0 else r.randint(max(1, c["context"] // 4), c["context"])
        new = c["new"]
        if c["mixed"] and b and r.random() < 0.7:
            new = 1
        elif new > 1 and b:
            new = r.randint(max(1, new // 2), new)
        out.append((n, min(n, new)))
    return out


def _axes(c):
    n = [x for x in (c["n1"], c["n2"], c["n3"]) if x]
    return n, [c["p1"], c["p2"], c["p3"]][:len(n)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(c, g, *shape):
    return torch.randn(shape, device="cuda", generator=g).to(_TYPES[c["dtype"]])


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "sliding":
        B, L, Cq, Ck = c["batch"], c["length"], c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
        # one projection's output in three parts, as a layer has them
        qkv = _randn(c, g, B, L, Cq + 2 * Ck)
        s["q"], s["k"], s["v"] = qkv.split([Cq, Ck, Ck], dim=-1)
        if c["train"]:
            s["q"], s["k"], s["v"] = (t.detach().requires_grad_(True) for t in (s["q"], s["k"], s["v"]))
            s["dy"] = _randn(c, g, B, L, Cq)
        s["lengths"] = torch.tensor(_signal_lengths(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
    elif c["op"] in ("paged", "append"):
        seqs = _sequences(c)
        need = [-(-n // c["page"]) for n, _ in seqs]
        width, total = max(need), sum(need)
        r = random.Random(seed)
        order = list(range(total + 3))
        r.shuffle(order)
        rows, at = [], 0
        for n in need:
            rows.append(order[at:at + n] + [-1] * (width - n))
            at += n
        s["pages"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        s["lengths"] = torch.tensor([n for n, _ in seqs], dtype=torch.int32, device="cuda")
        offs = [0]
        for _, new in seqs:
            offs.append(offs[-1] + new)
        s["offsets"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
        s["total"], s["most_new"] = offs[-1], max(new for _, new in seqs)
        Ck = c["kv_heads"] * c["dim"]
        s["cache_k"], s["cache_v"] = (_randn(c, g, total + 3, c["page"], Ck) for _ in range(2))
        rows = offs[-1] + c["pad"]
        if c["op"] == "paged":
            s["q"] = _randn(c, g, rows, c["heads"] * c["dim"])
        else:
            s["k"], s["v"] = _randn(c, g, rows, Ck), _randn(c, g, rows, Ck)
    else:
        n, _ = _axes(c)
        shape = (c["batch"], *reversed(n), c["heads"] * c["dim"])
        s["x"] = _randn(c, g, *shape)
        s["positions"] = None
        if c["given"]:
            # a grid that starts somewhere else for each axis, far along the first
            grid = torch.meshgrid(*(torch.arange(m, device="cuda", dtype=torch.int32) for m in reversed(n)), indexing="ij")
            first = torch.randint(0, 100000, (len(n),), device="cuda", generator=g, dtype=torch.int32)
            s["positions"] = torch.stack([t + f for t, f in zip(reversed(grid), first)], -1).contiguous()
        if c["train"]:
            s["x"].requires_grad_(True)
            s["dy"] = _randn(c, g, *shape)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _heads(x, heads):
    """(B, L, heads*D) -> (B, heads, L, D) in 32 bits."""
    return x.detach().float().reshape(*x.shape[:2], heads, -1).transpose(1, 2)


def _plain_sliding(s):
    c = s["case"]
    B, L, H, Hk, D = c["batch"], c["length"], c["heads"], c["kv_heads"], c["dim"]
    G, scale, dt = H // Hk, 1.0 / math.sqrt(D), s["q"].dtype
    i = torch.arange(L, device="cuda")
    see = (i[None, :] <= i[:, None]) & ((i[None, :] > i[:, None] - c["window"]) | (i[None, :] < c["sinks"]))
    live = torch.ones((B, L), dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        live = i[None, :] < s["lengths"][:, None]
    see = (see[None] & live[:, None, :] & live[:, :, None])[:, None, None]
    q = _heads(s["q"], H).reshape(B, Hk, G * L, D)
    k, v = _heads(s["k"], Hk), _heads(s["v"], Hk)
    p = (q @ k.transpose(-1, -2)).reshape(B, Hk, G, L, L).mul_(scale).masked_fill_(~see, -math.inf)
    p = torch.exp_(p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)))
    p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-37))
    p = p.reshape(B, Hk, G * L, L)
    y = p @ v

    def tokens(x, heads):
        return x.reshape(B, heads, L, D).transpose(1, 2).reshape(B, L, heads * D).to(dt)

    if not c["train"]:
        return tokens(y, H)
    dy = _heads(s["dy"], H).reshape(B, Hk, G * L, D)
    dv = p.transpose(-1, -2) @ dy
    ds = (dy @ v.transpose(-1, -2)).sub_((dy * y).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    return tokens(y, H), tokens(dq, H), tokens(dk, Hk), tokens(dv, Hk)


def _rows(s):
    """(sequence, number in its chunk, position) of every new token."""
    r = torch.arange(s["total"], device="cuda")
    offs = s["offsets"].long()
    b = torch.searchsorted(offs[1:], r, right=True)
    t = r - offs[b]
    return b, t, s["lengths"].long()[b] - (offs[b + 1] - offs[b]) + t


def _plain_paged(s):
    c = s["case"]
    B, H, Hk, D, n = c["batch"], c["heads"], c["kv_heads"], c["dim"], s["most_new"]
    G = H // Hk
    b, t, pos = _rows(s)
    table = s["pages"].clamp(min=0).long()
    k, v = (s[x][table].float().reshape(B, -1, Hk, D).transpose(1, 2) for x in ("cache_k", "cache_v"))
    q = torch.zeros((B, n, H, D), device="cuda")
    at = torch.full((B, n), -1, dtype=torch.int64, device="cuda")
    q[b, t] = s["q"][:s["total"]].float().reshape(-1, H, D)
    at[b, t] = pos
    q = q.reshape(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * n, D)
    j = torch.arange(k.shape[2], device="cuda")
    see = (j <= at[..., None]) & ((j > at[..., None] - c["window"]) | (j < c["sinks"]))
    p = (q @ k.transpose(-1, -2)).reshape(B, Hk, G, n, -1).mul_(1.0 / math.sqrt(D))
    p = p.masked_fill_(~see[:, None, None], -math.inf)
    p = torch.exp_(p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)))
    p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-37))
    y = (p.reshape(B, Hk, G * n, -1) @ v).reshape(B, Hk, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, H * D)
    out = torch.zeros_like(s["q"])
    out[:s["total"]] = y[b, t].to(out.dtype)
    return out


def _plain_append(s):
    page = s["case"]["page"]
    b, _, pos = _rows(s)
    slot = s["pages"].long()[b, pos // page] * page + pos % page
    for cache, new in ((s["cache_k"], s["k"]), (s["cache_v"], s["v"])):
        cache.view(-1, cache.shape[-1])[slot] = new[:s["total"]]
    return s["cache_k"], s["cache_v"]


_BASE = 10000.0


def _angles(c, positions):
    """cos and sin of every rotated pair, (1, *grid, 1, pairs): formed in 64
    bits, where far positions keep their angle."""
    n, p = _axes(c)
    parts = []
    for a, (size, pairs) in enumerate(zip(n, p)):
        if positions is None:
            shape = [1] * len(n)
            shape[len(n) - 1 - a] = size
            at = torch.arange(size, device="cuda", dtype=torch.float64).reshape(shape).expand(*reversed(n))
        else:
            at = positions[..., a].double()
        f = _BASE ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
        parts.append(at[..., None] * f)
    ang = torch.cat(parts, -1)[None, ..., None, :]
    return torch.cos(ang).float(), torch.sin(ang).float()


def _turn(c, x, cos, sin):
    """Every head's pairs turned by their angles; the channels behind stay."""
    h = x.detach().float().reshape(*x.shape[:-1], c["heads"], c["dim"])
    out, at, pair = h.clone(), 0, 0
    for p in _axes(c)[1]:
        if c["interleaved"]:
            i = torch.arange(p, device="cuda") * 2 + at
            j = i + 1
        else:
            i = torch.arange(p, device="cuda") + at
            j = i + p
        cs, sn = cos[..., pair:pair + p], sin[..., pair:pair + p]
        out[..., i], out[..., j] = h[..., i] * cs - h[..., j] * sn, h[..., i] * sn + h[..., j] * cs
        at, pair = at + 2 * p, pair + p
    return out.reshape(x.shape).to(x.dtype)


def _plain_rotary(s):
    cos, sin = _angles(s["case"], s["positions"])
    y = _turn(s["case"], s["x"], cos, sin)
    return (y, _turn(s["case"], s["dy"], cos, -sin)) if s["case"]["train"] else y


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _own(s):
    ca, c = _ca(), s["case"]
    if c["op"] == "sliding":
        call = {"kv_heads": c["kv_heads"], "sinks": c["sinks"], "lengths": s["lengths"]}
        if c["train"]:
            y = ca.sliding_mh_attention(s["q"], s["k"], s["v"], c["window"], c["heads"], **call)
            return (y.detach(), *torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["dy"]))
        with torch.no_grad():
            return ca.sliding_mh_attention(s["q"], s["k"], s["v"], c["window"], c["heads"], **call)
    if c["op"] == "paged":
        return ca.paged_mh_attention(s["q"], s["cache_k"], s["cache_v"], s["pages"], s["lengths"], c["window"], c["heads"],
                                     kv_heads=c["kv_heads"], sinks=c["sinks"],
                                     offsets=None if c["new"] == 1 and not c["pad"] else s["offsets"])
    if c["op"] == "append":
        ca.paged_append_(s["cache_k"], s["cache_v"], s["k"], s["v"], s["pages"], s["lengths"],
                         offsets=None if c["new"] == 1 and not c["pad"] else s["offsets"])
        return s["cache_k"], s["cache_v"]
    call = {"base": _BASE, "positions": s["positions"], "interleaved": c["interleaved"]}
    pairs = tuple(_axes(c)[1])
    if c["train"]:
        y = ca.axial_rotary(s["x"], pairs, c["heads"], **call)
        return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]
    with torch.no_grad():
        return ca.axial_rotary(s["x"], pairs, c["heads"], **call)


def run(state):
    if own:
        return _own(state)
    return {"sliding": _plain_sliding, "paged": _plain_paged, "append": _plain_append,
            "rotary": _plain_rotary}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _seen(first, last, c):
    """(sum over positions first..last of the keys seen, distinct keys read)."""
    most = c["window"] + c["sinks"]
    full = max(0, last - max(first, most) + 1)          # rows that see `most`
    a, b = first + 1, min(last, most - 1) + 1           # the others see a..b
    pairs = full * most + ((a + b) * (b - a + 1) // 2 if b >= a else 0)
    low = max(0, first - c["window"] + 1)
    return pairs, last + 1 - low + min(c["sinks"], low)


def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "sliding":
        pairs = sum(_seen(0, n - 1, c)[0] for n in _signal_lengths(c)) * c["heads"] * c["dim"]
        tokens = c["batch"] * c["length"]
        T = tokens * (2 * c["heads"] + 2 * c["kv_heads"]) * c["dim"] * e
        if c["train"]:  # and dy, dq, dk, dv
            return {"bytes": 2 * T, "flops": 14 * pairs}
        return {"bytes": T, "flops": 4 * pairs}
    if c["op"] == "paged":
        got = [_seen(n - new, n - 1, c) for n, new in _sequences(c)]
        rows = sum(new for _, new in _sequences(c))
        return {"bytes": (2 * rows * c["heads"] + 2 * sum(k for _, k in got) * c["kv_heads"]) * c["dim"] * e,
                "flops": 4 * sum(p for p, _ in got) * c["heads"] * c["dim"]}
    if c["op"] == "append":
        return {"bytes": 4 * sum(new for _, new in _sequences(c)) * c["kv_heads"] * c["dim"] * e, "flops": 0}
    n, p = _axes(c)
    tokens = c["batch"] * math.prod(n)
    k = 2 if c["train"] else 1
    given = 4 * math.prod(n) * len(n) if c["given"] else 0
    return {"bytes": k * (2 * tokens * c["heads"] * c["dim"] * e + given), "flops": k * 6 * tokens * c["heads"] * sum(p)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, a head at a time
# ---------------------------------------------------------------------------
def _exact_head(q, k, v, pos, c, dy=None):
    """One head: q (n, D) at positions pos over k, v (m, D)."""
    j = torch.arange(k.shape[0], device="cuda")
    d = pos[:, None] - j[None, :]
    hidden = (d < 0) | ((d >= c["window"]) & (j[None, :] >= c["sinks"]))
    a = torch.mm(q, k.t().contiguous()) / math.sqrt(q.shape[1])
    a[hidden] = -math.inf
    a = torch.softmax(a, 1)
    y = torch.mm(a, v)
    if dy is None:
        return y
    da = torch.mm(dy, v.t().contiguous())
    e = a * (da - (a * da).sum(1, keepdim=True)) / math.sqrt(q.shape[1])
    return y, torch.mm(e, k), torch.mm(e.t().contiguous(), q), torch.mm(a.t().contiguous(), dy)


def _exact_sliding(c, s):
    D, G = c["dim"], c["heads"] // c["kv_heads"]
    q, k, v = (s[x].detach().double() for x in "qkv")
    out = [torch.zeros_like(q)] + ([torch.zeros_like(t) for t in (q, k, v)] if c["train"] else [])
    for b, n in enumerate(_signal_lengths(c)):
        pos = torch.arange(n, device="cuda")
        for h in range(c["heads"]):
            hq, hk = slice(h * D, h * D + D), slice(h // G * D, h // G * D + D)
            x = (q[b, :n, hq], k[b, :n, hk], v[b, :n, hk])
            if not c["train"]:
                out[0][b, :n, hq] = _exact_head(*x, pos, c)
                continue
            y, dq, dk, dv = _exact_head(*x, pos, c, s["dy"].double()[b, :n, hq])
            out[0][b, :n, hq] = y
            out[1][b, :n, hq] = dq
            out[2][b, :n, hk] += dk
            out[3][b, :n, hk] += dv
    return tuple(out) if c["train"] else out[0]


def _exact_paged(c, s):
    D, G = c["dim"], c["heads"] // c["kv_heads"]
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, new) in enumerate(_sequences(c)):
        own_pages = s["pages"][b, :-(-n // c["page"])].long()
        k, v = (s[x].index_select(0, own_pages).flatten(0, 1)[:n].double() for x in ("cache_k", "cache_v"))
        pos = torch.arange(n - new, n, device="cuda")
        for h in range(c["heads"]):
            hq, hk = slice(h * D, h * D + D), slice(h // G * D, h // G * D + D)
            out[at:at + new, hq] = _exact_head(s["q"][at:at + new, hq].double(), k[:, hk], v[:, hk], pos, c)
        at += new
    return out


def _exact_append(c, s):
    k, v, at = s["cache_k"].double(), s["cache_v"].double(), 0
    for b, (n, new) in enumerate(_sequences(c)):
        pos = list(range(n - new, n))
        row = s["pages"][b].tolist()
        page = torch.tensor([row[p // c["page"]] for p in pos], device="cuda")
        slot = torch.tensor([p % c["page"] for p in pos], device="cuda")
        k[page, slot], v[page, slot] = s["k"][at:at + new].double(), s["v"][at:at + new].double()
        at += new
    return k, v


def _exact_rotary(c, s):
    n, p = _axes(c)

    def turned(x, sign):
        h = x.detach().double().reshape(*x.shape[:-1], c["heads"], c["dim"]).clone()
        at = 0
        for a, pairs in enumerate(p):
            f = torch.tensor([math.pow(_BASE, -i / pairs) for i in range(pairs)], dtype=torch.float64, device="cuda")
            if s["positions"] is None:
                where = torch.arange(n[a], device="cuda").reshape(-1, *[1] * a).expand(*reversed(n))
            else:
                where = s["positions"][..., a]
            w = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), sign * where.double()[..., None, None] * f)
            part = h[..., at:at + 2 * pairs]
            if c["interleaved"]:
                z = torch.view_as_complex(part.unflatten(-1, (pairs, 2)).contiguous()) * w
                h[..., at:at + 2 * pairs] = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(part[..., :pairs], part[..., pairs:]) * w
                h[..., at:at + 2 * pairs] = torch.cat([z.real, z.imag], -1)
            at += 2 * pairs
        return h.reshape(x.shape)

    return (turned(s["x"], 1.0), turned(s["dy"], -1.0)) if c["train"] else turned(s["x"], 1.0)


def exact(case, seed):
    s = prepare(case, seed)
    return {"sliding": _exact_sliding, "paged": _exact_paged, "append": _exact_append,
            "rotary": _exact_rotary}[case["op"]](case, s)
