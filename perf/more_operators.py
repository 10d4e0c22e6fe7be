"""Performance cases of the token attention with shaped scores (capped by a tanh,
biased by distance, masked by documents or by a prefix), for training and over a
paged cache, and of the cache's pages: sequences forked, resized and compacted.

A case is a dict of plain values; "op" says which operator:

  "sliding"  y = sliding_mh_attention(q, k, v, W, heads, cap=, slopes=, places=,
             prefix=); train: the gradients of q, k, v as well
  "paged"    y = paged_mh_attention(q, cache_k, cache_v, pages, lengths, W,
             heads, cap=, slopes=, prefix=): the new tokens of every sequence
  "resize"   paged_resize_(cache_k, cache_v, pages, lengths, counts, to): pages
             given and taken back, shared part pages copied before they are
             written; take: after paged_fork(pages, lengths, counts, source, page),
             with which sequences go on from others, whose pages they share
  "compact"  paged_compact_(cache_k, cache_v, pages, counts): pages moved to the
             lowest numbers

cap 0, documents 0 and prefix 0 mean none.  "spread" seeds the lengths, which belong
to the case; inputs and the order of the pages come from the seed of prepare().
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


def _sliding(name, batch, length, heads, kv_heads, dim, window, sinks, dtype, *, train=False, ragged=False, cap=0.0,
             slopes=False, documents=0, prefix=0, spread=0):
    return {"name": name, "op": "sliding", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "window": window, "sinks": sinks, "dtype": dtype, "train": train, "ragged": ragged, "cap": cap,
            "slopes": slopes, "documents": documents, "prefix": prefix, "spread": spread}


def _paged(name, batch, context, new, heads, kv_heads, dim, window, sinks, page, dtype, *, cap=0.0, slopes=False, prefix=0,
           mixed=False, spread=0):
    return {"name": name, "op": "paged", "batch": batch, "context": context, "new": new, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "page": page, "dtype": dtype, "cap": cap,
            "slopes": slopes, "prefix": prefix, "mixed": mixed, "spread": spread}


def _pages(name, op, batch, share, context, page, channels, dtype, *, take=0, grow=0, ended=0, spare=0, spread=0):
    """share: so many sequences each hold the same pages; take: sequences after a
    fork; grow, ended: tokens that a resize adds, per cent of the sequences that end;
    spare: per cent of the pool that nobody holds."""
    return {"name": name, "op": op, "batch": batch, "share": share, "context": context, "page": page,
            "channels": channels, "dtype": dtype, "take": take, "grow": grow, "ended": ended, "spare": spare,
            "spread": spread}


def listed():
    return [
        # a short signal of a small Float32 model with capped scores: latency
        _sliding("capped_small", 1, 77, 4, 4, 32, 32, 4, "f32", cap=20.0, slopes=True),
        # a long prompt through a layer with capped scores, no gradients
        _sliding("capped_prompt", 1, 8192, 32, 8, 128, 4096, 0, "bf16", cap=50.0),
        # a training step whose positions are a bias by distance
        _sliding("slopes_train", 2, 4096, 16, 4, 128, 1024, 0, "bf16", train=True, slopes=True),
        # packed documents of a training batch, odd lengths, capped scores
        _sliding("documents_train", 2, 4099, 12, 4, 80, 1 << 20, 0, "f16", train=True, cap=30.0, documents=600, spread=5),
        # a padded batch whose prefixes (an image's tokens, an instruction) see
        # themselves both ways
        _sliding("prefix_train", 3, 1531, 16, 8, 64, 512, 0, "bf16", train=True, ragged=True, prefix=576, spread=3),
        # the next token of a full serving batch, capped scores
        _paged("token_capped_batch", 64, 8192, 1, 32, 8, 128, 4096, 0, 16, "bf16", cap=50.0, spread=7),
        # chunks of prompts behind their prefixes, capped scores and a bias
        _paged("chunk_prefix", 4, 6000, 512, 32, 8, 128, 2048, 0, 64, "bf16", cap=50.0, slopes=True, prefix=700, spread=3),
        # two prompts become four sequences that bring a token each: latency
        _pages("beams_small", "resize", 2, 1, 300, 16, 256, "f32", take=4, grow=1, spare=30, spread=4),
        # a step of a search over beams: sequences go on from others and bring a token
        _pages("beams_batch", "resize", 64, 4, 4096, 16, 1024, "bf16", take=128, grow=1, spare=10, spread=9),
        # a turn of a serving batch: some sequences end, some are rolled back, the
        # others bring 512 tokens
        _pages("turn_batch", "resize", 256, 1, 2048, 16, 128, "bf16", grow=512, ended=20, spread=7),
        # the pools of a small and of a long-running server after sequences ended
        _pages("compact_small", "compact", 4, 1, 300, 16, 240, "f16", ended=50, spare=10, spread=2),
        _pages("compact_pool", "compact", 64, 1, 2048, 16, 1024, "bf16", ended=50, spare=10, spread=11),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# the most that a drawn case takes, by operator: the scores of the plain form
# (rows x keys x heads), or the values moved
_MOST = {"sliding": 32 * 8192 ** 2, "sliding_train": 2 * 16 * 4096 ** 2, "paged": 64 * 32 * 8192,
         "chunk": 4 * 32 * 512 * 6000, "pool": 64 * 2048 * 1024}


def draw(rng):
    """Signals of 1 to 8192 tokens, contexts of 1 to 16384, chunks of 1 to 1024,
    windows of 1 to everything, heads of 8 to 128 channels in groups of 1 to 8, caps
    of 5 to 100, documents of 1 to 2000 tokens, prefixes of 1 to everything, pools of
    1 to 256 sequences; all three types."""
    dtype = rng.choice(["bf16"] * 5 + ["f16"] * 3 + ["f32"] * 2)
    dim = rng.choice([8, 16, 32, 40, 64, 64, 72, 80, 96, 104, 128, 128, 128])
    kv_heads, group = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    window = rng.choice([_log_int(rng, 1, 8192), _log_int(rng, 32, 4096), 1 << 20])
    sinks = rng.choice([0, 0, 0, 1, 4, rng.randint(2, 64)])
    cap = rng.choice([0.0, 20.0, 30.0, 50.0, round(math.exp(rng.uniform(math.log(5), math.log(100))), 2)])
    slopes = rng.random() < 0.4
    spread = rng.randint(0, 1 << 20)
    op = rng.choice(["sliding"] * 5 + ["paged"] * 4 + ["resize"] * 2 + ["compact"])
    while True:
        if op == "sliding":
            train = rng.random() < 0.6
            length = _log_int(rng, 1, 8192)
            kind = rng.choice(["", "documents", "prefix"]) if cap or slopes else rng.choice(["documents", "prefix"])
            c = _sliding("", rng.choice([1, 1, 2, 3, 5]), length, kv_heads * group, kv_heads, dim, window, sinks, dtype,
                         train=train, ragged=rng.random() < 0.3, cap=cap, slopes=slopes,
                         documents=_log_int(rng, 1, 1000) if kind == "documents" else 0,
                         prefix=_log_int(rng, 1, length) if kind == "prefix" else 0, spread=spread)
            cost, most = c["batch"] * c["heads"] * c["length"] ** 2, _MOST["sliding_train" if train else "sliding"]
        elif op == "paged":
            one = rng.random() < 0.5
            context = _log_int(rng, 1, 16384)
            new = 1 if one else min(context, _log_int(rng, 1, 1024))
            prefix = _log_int(rng, 1, context) if rng.random() < 0.3 or not (cap or slopes) else 0
            c = _paged("", _log_int(rng, 1, 128 if one else 40), context, new, kv_heads * group, kv_heads, dim, window,
                       sinks, rng.choice([8, 16, 16, 32, 64, 128]), dtype, cap=cap, slopes=slopes, prefix=prefix,
                       mixed=not one and rng.random() < 0.5, spread=spread)
            cost = c["batch"] * c["heads"] * new * context
            # the plain form reads its caches in 32 bits; one token a sequence is bound by that
            cost, most = (cost * dim // 128, _MOST["paged"]) if one else (cost, _MOST["chunk"])
            if c["batch"] * context * kv_heads * dim > 64 * 8192 * 1024:
                continue
        else:
            batch, context, grow = _log_int(rng, 1, 256), _log_int(rng, 1, 8192), rng.choice([1, 1, _log_int(rng, 1, 2048)])
            take = _log_int(rng, 1, 256) if op == "resize" and rng.random() < 0.5 else 0
            c = _pages("", op, batch, rng.choice([1, 1, 2, 4, 8]), context, rng.choice([8, 16, 16, 32, 64]),
                       rng.choice([64, 128, 240, 512, 1024]), dtype, take=take, grow=grow if op == "resize" else 0,
                       ended=0 if take else rng.choice([0, 10, 50, 90]), spare=rng.choice([0, 5, 30, 60]), spread=spread)
            cost = (batch * context + (take or batch) * c["grow"]) * c["channels"] * (2 if dtype == "f32" else 1)
            most = _MOST["pool"]
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


def _documents(c):
    """The documents of every signal: their lengths, in order."""
    r = random.Random(c["spread"] + 1)
    out = []
    for _ in range(c["batch"]):
        left, got = c["length"], []
        while left > 0:
            got.append(min(left, r.randint(1, 2 * c["documents"])))
            left -= got[-1]
        out.append(got)
    return out


def _prefixes(c, lengths):
    r = random.Random(c["spread"] + 2)
    return [min(n, c["prefix"] if b == 0 else r.randint(0, c["prefix"])) for b, n in enumerate(lengths)]


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


def _held(c):
    """Of every sequence of a pool: its group (whose pages it shares), its tokens,
    and the tokens it is resized to (-1: as it is)."""
    r = random.Random(c["spread"])
    lengths = {}
    out = []
    for b in range(c["batch"]):
        g = b // c["share"]
        if g not in lengths:
            lengths[g] = c["context"] if g == 0 else r.randint(max(1, c["context"] // 4), c["context"])
        n, dice = lengths[g], r.random() * 100
        if c["op"] == "compact":  # those that ended are gone
            to = 0 if dice < c["ended"] else n
        elif dice < c["ended"]:
            to = 0
        elif dice > 95 and c["grow"] > 1:
            to = -1 if dice > 97 else r.randint(0, n)  # waits, or is rolled back
        else:
            to = n + c["grow"]
        out.append((g, n, to))
    return out


def _pool(c, seed):
    """(rows of the table, tokens, counts of holders, tokens wanted) as lists."""
    seqs, page = _held(c), c["page"]
    need = {g: -(-n // page) for g, n, _ in seqs}
    total = sum(need.values())
    more = sum(max(0, -(-to // page) - -(-n // page) + 1) for _, n, to in seqs if to > n)
    more = max(more, c["take"] * (-(-c["grow"] // page) + 1))
    npages = max(1, total + (more if c["op"] == "resize" else 0))
    npages += npages * c["spare"] // 100
    order = list(range(npages))
    random.Random(seed).shuffle(order)
    own_pages, at = {}, 0
    for g in need:
        own_pages[g] = order[at:at + need[g]]
        at += need[g]
    width = max(1, max(-(-(max(n, to) + (c["grow"] if c["take"] else 0)) // page) for _, n, to in seqs))
    counts, rows, lengths = [0] * npages, [], []
    for g, n, to in seqs:
        if c["op"] == "compact" and to == 0:
            rows.append([-1] * width)
            lengths.append(0)
            continue
        for p in own_pages[g]:
            counts[p] += 1
        rows.append(own_pages[g] + [-1] * (width - need[g]))
        lengths.append(n)
    return rows, lengths, counts, [to for _, _, to in seqs]


def _source(c, seed):
    """Where a fork's sequences come from; a few places stay empty."""
    r = random.Random(seed + 1)
    return [-1 if r.random() < 0.03 else r.randrange(c["batch"]) for _ in range(c["take"])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(c, g, *shape):
    return torch.randn(shape, device="cuda", generator=g).to(_TYPES[c["dtype"]])


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _slopes(c):
    """A geometric sequence over the heads, from 2^(-8/H) down to 2^-8."""
    h = torch.arange(1, c["heads"] + 1, device="cuda", dtype=torch.float64)
    return torch.exp2(-8.0 * h / c["heads"]).float() if c["slopes"] else None


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    # where scores are capped they are large enough for the cap to matter
    loud = 3.0 if c.get("cap") else 1.0
    if c["op"] == "sliding":
        B, L, Cq, Ck = c["batch"], c["length"], c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
        # one projection's output in three parts, as a layer has them
        qkv = _randn(c, g, B, L, Cq + 2 * Ck)
        qkv[..., :Cq] *= loud
        s["q"], s["k"], s["v"] = qkv.split([Cq, Ck, Ck], dim=-1)
        if c["train"]:
            s["q"], s["k"], s["v"] = (t.detach().requires_grad_(True) for t in (s["q"], s["k"], s["v"]))
            s["dy"] = _randn(c, g, B, L, Cq)
        lengths = _signal_lengths(c)
        s["lengths"] = _ints(lengths) if c["ragged"] else None
        s["slopes"] = _slopes(c)
        s["places"] = s["prefix"] = None
        if c["documents"]:
            s["places"] = torch.stack([torch.cat([torch.arange(n, dtype=torch.int32) for n in d])
                                       for d in _documents(c)]).cuda()
        if c["prefix"]:
            s["prefix"] = _ints(_prefixes(c, lengths))
        return s
    if c["op"] == "paged":
        seqs = _sequences(c)
        need = [-(-n // c["page"]) for n, _ in seqs]
        width, total = max(need), sum(need)
        order = list(range(total + 3))
        random.Random(seed).shuffle(order)
        rows, at = [], 0
        for n in need:
            rows.append(order[at:at + n] + [-1] * (width - n))
            at += n
        offs = [0]
        for _, new in seqs:
            offs.append(offs[-1] + new)
        s["pages"], s["lengths"], s["offsets"] = _ints(rows), _ints([n for n, _ in seqs]), _ints(offs)
        s["total"], s["most_new"] = offs[-1], max(new for _, new in seqs)
        Ck = c["kv_heads"] * c["dim"]
        s["cache_k"], s["cache_v"] = (_randn(c, g, total + 3, c["page"], Ck) for _ in range(2))
        s["q"] = _randn(c, g, offs[-1], c["heads"] * c["dim"]) * loud
        s["slopes"] = _slopes(c)
        s["prefix"] = _ints(_prefixes(c, [n for n, _ in seqs])) if c["prefix"] else None
        return s
    rows, lengths, counts, to = _pool(c, seed)
    s["pages"], s["lengths"], s["counts"] = _ints(rows), _ints(lengths), _ints(counts)
    if c["take"]:
        s["source"] = _ints(_source(c, seed))
    s["to"] = _ints(to)
    s["cache_k"], s["cache_v"] = (_randn(c, g, len(counts), c["page"], c["channels"]) for _ in range(2))
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _heads(x, heads):
    """(B, L, heads*D) -> (B, heads, L, D) in 32 bits."""
    return x.detach().float().reshape(*x.shape[:2], heads, -1).transpose(1, 2)


def _plain_scores(c, x, far, slopes):
    """Capped and biased in place; x: (B, Hk, G, rows, keys), far: their distances."""
    if c["cap"]:
        x.div_(c["cap"]).tanh_().mul_(c["cap"])
    if slopes is not None:
        x.addcmul_(far, -slopes.reshape(c["kv_heads"], -1, 1, 1))
    return x


def _plain_softmax(x, see):
    x = x.masked_fill_(~see, -math.inf)
    x = torch.exp_(x.sub_(x.amax(-1, keepdim=True).clamp_(min=-3e38)))
    return x.div_(x.sum(-1, keepdim=True).clamp_(min=1e-37))


def _plain_sliding(s):
    c = s["case"]
    B, L, H, Hk, D = c["batch"], c["length"], c["heads"], c["kv_heads"], c["dim"]
    G, scale, dt = H // Hk, 1.0 / math.sqrt(D), s["q"].dtype
    i = torch.arange(L, device="cuda")
    first = torch.zeros((B, L), dtype=torch.int64, device="cuda") if s["places"] is None else i - s["places"]
    row, key, first = i[None, :, None], i[None, None, :], first[:, :, None]
    see = (key >= first) & (key <= row) & ((key > row - c["window"]) | (key < first + c["sinks"]))
    if s["prefix"] is not None:
        see = see | (key < s["prefix"][:, None, None])
    if s["lengths"] is not None:
        n = s["lengths"][:, None, None]
        see = see & (row < n) & (key < n)
    see = see[:, None, None]
    far = (row - key).abs().float()
    q = _heads(s["q"], H).reshape(B, Hk, G * L, D)
    k, v = _heads(s["k"], Hk), _heads(s["v"], Hk)
    p = (q @ k.transpose(-1, -2)).reshape(B, Hk, G, L, L).mul_(scale)
    slope = None
    if c["train"] and c["cap"]:
        slope = torch.tanh(p / c["cap"]).square_().neg_().add_(1.0).reshape(B, Hk, G * L, L)
    p = _plain_softmax(_plain_scores(c, p, far, s["slopes"]), see).reshape(B, Hk, G * L, L)
    y = p @ v

    def tokens(x, heads):
        return x.reshape(B, heads, L, D).transpose(1, 2).reshape(B, L, heads * D).to(dt)

    if not c["train"]:
        return tokens(y, H)
    dy = _heads(s["dy"], H).reshape(B, Hk, G * L, D)
    dv = p.transpose(-1, -2) @ dy
    ds = (dy @ v.transpose(-1, -2)).sub_((dy * y).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    if slope is not None:
        ds.mul_(slope)
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
    if s["prefix"] is not None:
        see = see | ((j < s["prefix"][:, None, None]) & (at[..., None] >= 0))
    far = (at[:, None, None, :, None] - j).abs().float()
    x = (q @ k.transpose(-1, -2)).reshape(B, Hk, G, n, -1).mul_(1.0 / math.sqrt(D))
    p = _plain_softmax(_plain_scores(c, x, far, s["slopes"]), see[:, None, None])
    y = (p.reshape(B, Hk, G * n, -1) @ v).reshape(B, Hk, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, H * D)
    return y[b, t].to(s["q"].dtype)


def _there(pages, lengths, npages, page):
    """(entries that a sequence's tokens reach, those that are pages of the cache)."""
    e = torch.arange(pages.shape[1], device="cuda")
    reached = e < ((lengths.long().clamp(min=0) + page - 1) // page)[:, None]
    return reached, reached & (pages >= 0) & (pages < npages)


def _plain_fork(s):
    pages, lengths, counts, source = s["pages"], s["lengths"], s["counts"], s["source"].long()
    npages = counts.numel()
    some = (source >= 0) & (source < pages.shape[0])
    source = source.clamp(0, pages.shape[0] - 1)
    reached, there = _there(pages, lengths, npages, s["case"]["page"])
    new_pages = torch.where(reached[source] & some[:, None], pages[source], -1)
    new_lengths = torch.where(some, lengths[source], 0)
    new_there = there[source] & some[:, None]
    new_counts = counts.clone()
    for table, real, sign in ((pages, there, -1), (new_pages, new_there, 1)):
        where = torch.where(real, table, 0).long().flatten()
        new_counts.scatter_add_(0, where, (real.int() * sign).flatten())
    return new_pages, new_lengths, new_counts


def _plain_resize(s):
    pages, lengths, counts, to, page = s["pages"], s["lengths"], s["counts"], s["to"], s["case"]["page"]
    forked = ()
    if s["case"]["take"]:
        forked = pages, lengths, counts = _plain_fork(s)
        to = lengths + s["case"]["grow"]
    npages, width = counts.numel(), pages.shape[1]
    n = lengths.long().clamp(0, width * page)
    to = torch.where(to < 0, n, to.long().clamp(max=width * page))
    has, wants = (n + page - 1) // page, (to + page - 1) // page
    e = torch.arange(width, device="cuda")
    real = (pages >= 0) & (pages < npages)
    gone = (e >= wants[:, None]) & (e < has[:, None]) & real
    counts = counts.clone().scatter_add_(0, torch.where(gone, pages, 0).long().flatten(), -gone.int().flatten())
    # a part page that others hold is copied before it is written
    last = pages.gather(1, (has - 1).clamp(min=0)[:, None])[:, 0].long()
    last_real = (last >= 0) & (last < npages) & (has > 0)
    last = last.clamp(0, npages - 1)
    copied = (to > n) & (n % page != 0) & last_real & (counts[last] > 1)
    need = copied.long() + (wants - has).clamp(min=0)
    end = need.cumsum(0)
    free = counts == 0
    served = (need == 0) | (end <= free.sum())
    to, wants = torch.where(served, to, n), torch.where(served, wants, has)
    copied = copied & served
    numbers = torch.full((npages + 1,), -1, dtype=torch.int64, device="cuda")
    numbers.scatter_(0, torch.where(free, free.long().cumsum(0) - 1, npages), torch.arange(npages, device="cuda"))
    numbers[npages] = -1
    first = end - need
    given = (e >= has[:, None]) & (e < wants[:, None])
    rank = (first + copied)[:, None] + e - has[:, None]
    out = torch.where(given, numbers[rank.clamp(0, npages)], pages.long())
    fresh = numbers[first.clamp(0, npages)]
    is_last = copied[:, None] & (e == (has - 1)[:, None])
    out = torch.where(is_last, fresh[:, None], out)
    out = torch.where(e < wants[:, None], out, -1)
    counts.scatter_add_(0, last, -copied.int())
    taken = given | is_last
    counts.scatter_add_(0, torch.where(taken, out, 0).flatten(), taken.int().flatten())
    token = torch.arange(page, device="cuda")
    move = (copied[:, None] & (token < (n % page)[:, None])).flatten()
    whence = (last[:, None] * page + token).flatten()[move]
    whither = (fresh[:, None] * page + token).flatten()[move]
    for x in ("cache_k", "cache_v"):
        flat = s[x].view(npages * page, -1)
        flat[whither] = flat[whence]
    return (*forked, out.int(), to.int(), counts, s["cache_k"], s["cache_v"])


def _plain_compact(s):
    pages, counts = s["pages"], s["counts"]
    npages = counts.numel()
    number = torch.arange(npages, device="cuda")
    used = counts > 0
    most = used.sum()
    movers, holes = (used & (number >= most)).nonzero()[:, 0], (~used & (number < most)).nonzero()[:, 0]
    where = number.clone()
    where[movers] = holes
    out_counts = counts.clone()
    out_counts[holes] = counts[movers]
    out_counts[movers] = 0
    real = (pages >= 0) & (pages < npages)
    out = torch.where(real, where[pages.clamp(0, npages - 1).long()].int(), pages)
    for x in ("cache_k", "cache_v"):
        s[x][holes] = s[x][movers]
    return out, out_counts, s["cache_k"], s["cache_v"]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _own(s):
    ca, c = _ca(), s["case"]
    if c["op"] == "sliding":
        call = {"kv_heads": c["kv_heads"], "sinks": c["sinks"], "lengths": s["lengths"], "cap": c["cap"] or None,
                "slopes": s["slopes"], "places": s["places"], "prefix": s["prefix"]}
        if c["train"]:
            y = ca.sliding_mh_attention(s["q"], s["k"], s["v"], c["window"], c["heads"], **call)
            return (y.detach(), *torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["dy"]))
        with torch.no_grad():
            return ca.sliding_mh_attention(s["q"], s["k"], s["v"], c["window"], c["heads"], **call)
    if c["op"] == "paged":
        return ca.paged_mh_attention(s["q"], s["cache_k"], s["cache_v"], s["pages"], s["lengths"], c["window"], c["heads"],
                                     kv_heads=c["kv_heads"], sinks=c["sinks"], cap=c["cap"] or None, slopes=s["slopes"],
                                     prefix=s["prefix"], offsets=None if c["new"] == 1 else s["offsets"])
    if c["op"] == "resize":
        table, to, forked = (s["pages"], s["lengths"], s["counts"]), s["to"], ()
        if c["take"]:
            forked = table = ca.paged_fork(*table, s["source"], c["page"])
            to = table[1] + c["grow"]
        return (*forked, *ca.paged_resize_(s["cache_k"], s["cache_v"], *table, to), s["cache_k"], s["cache_v"])
    return (*ca.paged_compact_(s["cache_k"], s["cache_v"], s["pages"], s["counts"]), s["cache_k"], s["cache_v"])


def run(state):
    if own:
        return _own(state)
    return {"sliding": _plain_sliding, "paged": _plain_paged, "resize": _plain_resize,
            "compact": _plain_compact}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _seen(first, last, c, prefix=0):
    """(sum over positions first..last of a sequence of the keys seen, distinct keys
    read)."""
    pairs = 0
    for i in range(first, last + 1):
        low = max(0, i - c["window"] + 1)
        ahead = max(prefix, min(c["sinks"], i + 1))   # seen from the start on
        pairs += i + 1 if ahead >= low else ahead + i + 1 - low
        pairs += max(0, prefix - i - 1)               # and behind itself
    low = max(0, first - c["window"] + 1)
    return pairs, max(last + 1, prefix) - low + min(max(c["sinks"], prefix), low)


def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "sliding":
        lengths = _signal_lengths(c)
        if c["documents"]:
            pairs = 0
            for n, docs in zip(lengths, _documents(c)):
                at = 0
                for d in docs:
                    got = max(0, min(d, n - at))
                    pairs += _seen(0, got - 1, c)[0] if got else 0
                    at += d
        else:
            prefix = _prefixes(c, lengths) if c["prefix"] else [0] * c["batch"]
            pairs = sum(_seen(0, n - 1, c, p)[0] if n else 0 for n, p in zip(lengths, prefix))
        pairs *= c["heads"] * c["dim"]
        tokens = c["batch"] * c["length"]
        T = tokens * (2 * c["heads"] + 2 * c["kv_heads"]) * c["dim"] * e
        if c["train"]:  # and dy, dq, dk, dv
            return {"bytes": 2 * T, "flops": 14 * pairs}
        return {"bytes": T, "flops": 4 * pairs}
    if c["op"] == "paged":
        seqs = _sequences(c)
        prefix = _prefixes(c, [n for n, _ in seqs]) if c["prefix"] else [0] * c["batch"]
        got = [_seen(n - new, n - 1, c, p) for (n, new), p in zip(seqs, prefix)]
        rows = sum(new for _, new in seqs)
        return {"bytes": (2 * rows * c["heads"] + 2 * sum(k for _, k in got) * c["kv_heads"]) * c["dim"] * e,
                "flops": 4 * sum(p for p, _ in got) * c["heads"] * c["dim"]}
    rows, lengths, counts, to = _pool(c, 0)
    page, width, token = c["page"], len(rows[0]), c["channels"] * e * 4  # k and v, read and written
    around = 0
    if c["take"]:
        # the table read and the new one written, lengths, and the counts twice
        around = 4 * width * (c["batch"] + c["take"]) + 4 * c["batch"] + 8 * c["take"] + 8 * len(counts)
        rows, lengths, counts = _forked(c, 0, rows, lengths, counts)
        to = [n + c["grow"] for n in lengths]
    around += 8 * len(rows) * width + 8 * len(counts) + 12 * len(rows)
    if c["op"] == "resize":
        part = sum(n % page for row, n, t in zip(rows, lengths, to) if t > n and n % page and counts[row[n // page]] > 1)
        return {"bytes": around + part * token, "flops": 0}
    most = sum(x > 0 for x in counts)
    moved = sum(x > 0 for x in counts[most:])
    return {"bytes": around + moved * page * token, "flops": 0}


# ---------------------------------------------------------------------------
# the definitions in 64 bits: attention a head at a time, pages a sequence at a time
# ---------------------------------------------------------------------------
def _exact_head(q, k, v, hidden, back, c, slope, dy=None):
    """One head: q (n, D) over k, v (m, D); back (n, m): how far a key lies back."""
    x = torch.mm(q, k.t().contiguous()) / math.sqrt(q.shape[1])
    bent = None
    if c["cap"]:
        t = torch.tanh(x / c["cap"])
        x, bent = t * c["cap"], 1 - t * t
    if slope is not None:
        x = x - slope * back.abs()
    a = torch.softmax(x.masked_fill(hidden, -math.inf), 1)
    y = torch.mm(a, v)
    if dy is None:
        return y
    da = torch.mm(dy, v.t().contiguous())
    e = a * (da - (a * da).sum(1, keepdim=True)) / math.sqrt(q.shape[1])
    if bent is not None:
        e = e * bent
    return y, torch.mm(e, k), torch.mm(e.t().contiguous(), q), torch.mm(a.t().contiguous(), dy)


def _hidden(c, back, key, prefix=0):
    return ((back < 0) | ((back >= c["window"]) & (key >= c["sinks"]))) & (key >= prefix)


def _exact_sliding(c, s):
    D, G = c["dim"], c["heads"] // c["kv_heads"]
    q, k, v = (s[x].detach().double() for x in "qkv")
    out = [torch.zeros_like(q)] + ([torch.zeros_like(t) for t in (q, k, v)] if c["train"] else [])
    dy = s["dy"].double() if c["train"] else None
    slopes = None if s["slopes"] is None else s["slopes"].double().tolist()
    lengths = _signal_lengths(c)
    prefix = _prefixes(c, lengths) if c["prefix"] else [0] * c["batch"]
    # every document by itself
    docs = _documents(c) if c["documents"] else [[n] for n in lengths]
    for b, n in enumerate(lengths):
        at = 0
        for d in docs[b]:
            end = min(at + d, n)
            if end > at:
                pos = torch.arange(end - at, device="cuda")
                back = pos[:, None] - pos[None, :]
                hidden = _hidden(c, back, pos[None, :], prefix[b])
                for h in range(c["heads"]):
                    hq, hk = slice(h * D, h * D + D), slice(h // G * D, h // G * D + D)
                    x = (q[b, at:end, hq], k[b, at:end, hk], v[b, at:end, hk], hidden, back, c, slopes and slopes[h])
                    if not c["train"]:
                        out[0][b, at:end, hq] = _exact_head(*x)
                        continue
                    y, dq, dk, dv = _exact_head(*x, dy[b, at:end, hq])
                    out[0][b, at:end, hq] = y
                    out[1][b, at:end, hq] = dq
                    out[2][b, at:end, hk] += dk
                    out[3][b, at:end, hk] += dv
            at += d
    return tuple(out) if c["train"] else out[0]


def _exact_paged(c, s):
    D, G = c["dim"], c["heads"] // c["kv_heads"]
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    slopes = None if s["slopes"] is None else s["slopes"].double().tolist()
    seqs = _sequences(c)
    prefix = _prefixes(c, [n for n, _ in seqs]) if c["prefix"] else [0] * c["batch"]
    for b, (n, new) in enumerate(seqs):
        own_pages = s["pages"][b, :-(-n // c["page"])].long()
        k, v = (s[x].index_select(0, own_pages).flatten(0, 1)[:n].double() for x in ("cache_k", "cache_v"))
        key = torch.arange(n, device="cuda")
        back = key[n - new:, None] - key[None, :]
        hidden = _hidden(c, back, key[None, :], prefix[b])
        for h in range(c["heads"]):
            hq, hk = slice(h * D, h * D + D), slice(h // G * D, h // G * D + D)
            out[at:at + new, hq] = _exact_head(s["q"][at:at + new, hq].double(), k[:, hk], v[:, hk], hidden, back, c,
                                               slopes and slopes[h])
        at += new
    return out


def _forked(c, seed, rows, lengths, counts):
    out_rows, out_lengths, width, counts = [], [], len(rows[0]), list(counts)
    for row, n in zip(rows, lengths):
        for p in row[:-(-n // c["page"])]:
            counts[p] -= 1
    for b in _source(c, seed):
        held = rows[b][:-(-lengths[b] // c["page"])] if b >= 0 else []
        for p in held:
            counts[p] += 1
        out_rows.append(held + [-1] * (width - len(held)))
        out_lengths.append(lengths[b] if b >= 0 else 0)
    return out_rows, out_lengths, counts


def _exact_resize(c, seed, s):
    rows, lengths, counts, to = _pool(c, seed)
    forked = ()
    if c["take"]:
        rows, lengths, counts = _forked(c, seed, rows, lengths, counts)
        forked = _ints(rows), _ints(lengths), _ints(counts)
        to = [n + c["grow"] for n in lengths]
    page = c["page"]
    to = [n if t < 0 else t for n, t in zip(lengths, to)]
    for row, n, t in zip(rows, lengths, to):
        for e in range(-(-t // page), -(-n // page)):
            counts[row[e]] -= 1
            row[e] = -1
    free = [p for p, x in enumerate(counts) if x == 0]
    shared = [x > 1 for x in counts]
    used, copies = 0, []
    for b, (row, n, t) in enumerate(zip(rows, lengths, to)):
        if t <= n:
            continue
        has, wants = -(-n // page), -(-t // page)
        copy = n % page != 0 and shared[row[has - 1]]
        used += wants - has + copy
        if wants - has + copy > 0 and used > len(free):
            to[b] = n
            continue
        mine = free[used - (wants - has) - copy:used]
        if copy:
            copies.append((row[has - 1], mine[0], n % page))
            counts[row[has - 1]] -= 1
            row[has - 1] = mine.pop(0)
            counts[row[has - 1]] = 1
        for e in range(has, wants):
            row[e] = mine.pop(0)
            counts[row[e]] = 1
    caches = []
    for x in ("cache_k", "cache_v"):
        cache = s[x].double()
        for a, b, m in copies:
            cache[b, :m] = s[x][a, :m].double()
        caches.append(cache)
    return *forked, _ints(rows), _ints(to), _ints(counts), *caches


def _exact_compact(c, seed, s):
    rows, _, counts, _ = _pool(c, seed)
    most = sum(x > 0 for x in counts)
    holes = [p for p in range(most) if counts[p] == 0]
    movers = [p for p in range(most, len(counts)) if counts[p] > 0]
    where = dict(zip(movers, holes))
    caches = [s[x].double() for x in ("cache_k", "cache_v")]
    for a, b in where.items():
        counts[b], counts[a] = counts[a], 0
        for cache, x in zip(caches, ("cache_k", "cache_v")):
            cache[b] = s[x][a].double()
    return _ints([[where.get(p, p) for p in row] for row in rows]), _ints(counts), *caches


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "resize":
        return _exact_resize(case, seed, s)
    if case["op"] == "compact":
        return _exact_compact(case, seed, s)
    return {"sliding": _exact_sliding, "paged": _exact_paged}[case["op"]](case, s)
