"""Downstream layers over the circulant attention entry points, in the manner
of GroupCDL (the reference's README.md:33-38 points to it as the example
consumer): an attention block for channels-last feature maps, and the
group-sparse thresholding whose group norms are circulant-attention sums; and
the attention block of a token model, with its serving step.

The first two take channels-last tensors (B, *spatial_slow_first, C), the layout of
`torch.nn.Linear` over the channel axis, so 1x1 projections need no
transposes and the fused kernels read the tensors in place
(`CIRCATT_CHANNELS_LAST`).  A spatial size (H, W) here is the reference's
Julia (W, H): the last spatial axis before C is the fastest.
"""
from __future__ import annotations

import torch

from .circulant import (AbstractSimilarity, Circulant, DistanceSimilarity, DotSimilarity,
                        Otimes, circulant_mh_adjacency, circulant_mh_attention)
from .tokens import axial_rotary, paged_append_, paged_mh_attention, sliding_mh_attention


class CircAttBlock(torch.nn.Module):
    """x + W_o · MHA(W_q x, W_k x, W_v x) with circulant (windowed, circularly
    wrapped) multi-head attention of window `window` over the spatial axes.

    x: (B, *spatial, channels), channels-last.  The attention is the fused
    path of circulant_mh_attention (src/attention.jl:38-42, A never formed)
    with the similarity `simfun` honoured; its scale is the reference's
    1/sqrt(channels per head).  `rotary`, one number of pairs for each spatial
    axis (fastest first), turns queries and keys with their pixel's position
    (axial_rotary); positions do not wrap, so a window over the border sees its
    pixels' positions as they are."""

    def __init__(self, channels: int, window: int, nheads: int = 1,
                 simfun: AbstractSimilarity = DotSimilarity(), bias: bool = True, rotary=None):
        super().__init__()
        if channels % nheads != 0:
            raise AssertionError(f"channels ({channels}) must be divisible by nheads ({nheads})")
        if window % 2 != 1:
            raise AssertionError(f"filter size M={window} must be odd.")
        self.window, self.nheads, self.simfun = window, nheads, simfun
        self.rotary = None if rotary is None else tuple(rotary)
        # separate projections: each output is a contiguous channels-last tensor
        self.q = torch.nn.Linear(channels, channels, bias=bias)
        self.k = torch.nn.Linear(channels, channels, bias=bias)
        self.v = torch.nn.Linear(channels, channels, bias=bias)
        self.o = torch.nn.Linear(channels, channels, bias=bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        q, k = self.q(x), self.k(x)
        if self.rotary is not None:
            q, k = (axial_rotary(t, self.rotary, self.nheads) for t in (q, k))
        y, _ = circulant_mh_attention(self.simfun, q, k, self.v(x), self.window,
                                      self.nheads, materialize=False, honor_simfun=True,
                                      channels_last=True)
        return x + self.o(y)


class SlidingAttBlock(torch.nn.Module):
    """x + W_o · SWA(rot(W_q x), rot(W_k x), W_v x) on token signals (B, L,
    channels): causal attention in a sliding window with sinks
    (sliding_mh_attention), nheads heads of queries over kv_heads of keys and
    values, and rotary positions with `rotary` = (pairs, ...) pairs for each axis
    (None: no positions).  `cap` bounds the scores, and with `distance` they fall by
    2^(-8 (h + 1) / nheads) a token of distance in head h (`slopes`, a buffer).

    `forward` is for training and whole prompts; `step` takes the new tokens of
    several sequences, appends their keys and values to a paged cache and
    attends over it.  A signal given to `step` in pieces has the rows that
    `forward` gives for the whole."""

    def __init__(self, channels: int, window: int, nheads: int = 1, kv_heads: int = None, sinks: int = 0,
                 rotary=None, base: float = 10000.0, bias: bool = True, cap: float = None, distance: bool = False):
        super().__init__()
        kv_heads = nheads if kv_heads is None else kv_heads
        if nheads < 1 or channels % nheads != 0:
            raise AssertionError(f"channels ({channels}) must be divisible by nheads ({nheads})")
        if kv_heads < 1 or nheads % kv_heads != 0:
            raise AssertionError(f"nheads ({nheads}) must be divisible by kv_heads ({kv_heads})")
        self.window, self.sinks, self.nheads, self.kv_heads = window, sinks, nheads, kv_heads
        self.rotary, self.base = None if rotary is None else tuple(rotary), base
        self.cap = cap
        self.register_buffer("slopes", self._slopes() if distance else None, persistent=False)
        self.parts = [channels, channels // nheads * kv_heads, channels // nheads * kv_heads]
        # one projection: the attention reads its three parts in place
        self.qkv = torch.nn.Linear(channels, sum(self.parts), bias=bias)
        self.o = torch.nn.Linear(channels, channels, bias=bias)

    def _slopes(self):
        h = torch.arange(1, self.nheads + 1, dtype=torch.float64, device="cpu")
        return torch.exp2(-8.0 * h / self.nheads).float()

    def _apply(self, fn, *args, **kwargs):
        # the slopes stay Float32 in a block of another type
        slopes = self.slopes
        out = super()._apply(fn, *args, **kwargs)
        if slopes is not None:
            at = self.slopes.device
            self.slopes = (self._slopes() if slopes.is_meta and at.type != "meta" else slopes).to(at)
        return out

    def _project(self, x, positions):
        q, k, v = self.qkv(x).split(self.parts, dim=-1)
        if self.rotary is not None:
            q = axial_rotary(q, self.rotary, self.nheads, base=self.base, positions=positions)
            k = axial_rotary(k, self.rotary, self.kv_heads, base=self.base, positions=positions)
        return q, k, v

    def forward(self, x: torch.Tensor, lengths: torch.Tensor = None, positions: torch.Tensor = None,
                places: torch.Tensor = None, prefix: torch.Tensor = None) -> torch.Tensor:
        """positions (int32, (L, axes) or (B, L, axes)): None for one axis that
        counts the tokens, of their document where places are given.  places, prefix:
        as sliding_mh_attention takes them."""
        if places is not None and positions is None and self.rotary is not None and len(self.rotary) == 1:
            positions = places[..., None]
        q, k, v = self._project(x, positions)
        y = sliding_mh_attention(q, k, v, self.window, self.nheads, kv_heads=self.kv_heads, sinks=self.sinks,
                                 lengths=lengths, cap=self.cap, slopes=self.slopes, places=places, prefix=prefix)
        return x + self.o(y)

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, pages: torch.Tensor,
             lengths: torch.Tensor, offsets: torch.Tensor = None, positions: torch.Tensor = None,
             prefix: torch.Tensor = None) -> torch.Tensor:
        """x: (T, channels), the new tokens; the other arguments as
        paged_mh_attention takes them.  positions (int32, (T, axes)): None, with
        one new token a sequence and one axis, for each token's place."""
        if self.rotary is not None and positions is None:
            if offsets is not None or len(self.rotary) != 1:
                raise AssertionError("positions are needed with offsets or several axes")
            positions = (lengths - 1)[:, None]
        q, k, v = self._project(x, positions)
        paged_append_(cache_k, cache_v, k, v, pages, lengths, offsets=offsets)
        y = paged_mh_attention(q, cache_k, cache_v, pages, lengths, self.window, self.nheads, kv_heads=self.kv_heads,
                               sinks=self.sinks, offsets=offsets, cap=self.cap, slopes=self.slopes, prefix=prefix)
        return x + self.o(y)


class GroupThresholding(torch.nn.Module):
    """GroupCDL-style group-sparse thresholding of codes z (B, *spatial, M):

        Γ = rowsoftmax(simfun(θ_i, θ_j)) over the circulant window, per head
            of M / nheads channels, with θ = W_θ f a projection of features f;
        ξ = Γ ⨷ z²                      (non-local group energies)
        z ← z · relu(1 − τ / sqrt(ξ + ε))  (τ > 0 per channel)

    Γ is the reference's circulant_mh_adjacency (unscaled similarity,
    src/similarity.jl:144-161, src/attention.jl:46-51) and ξ its ⨷.  With
    `fused=True` (default) ξ comes from the fused attention kernels on the
    channels-last tensors, Γ never formed: attention scales q and k by
    dh^(-1/4) each (src/attention.jl:20-21), so θ enters as θ dh^(1/4).
    `adjacency(f)` returns Γ as a Circulant (planar, materialised) for callers
    that reuse it over several iterations, as GroupCDL does; `forward(z, f,
    A=Γ)` then applies it."""

    def __init__(self, channels: int, feat_channels: int, window: int, nheads: int = 1,
                 simfun: AbstractSimilarity = DistanceSimilarity(), tau: float = 0.1,
                 eps: float = 1e-6, fused: bool = True):
        super().__init__()
        if channels % nheads != 0:
            raise AssertionError(f"channels ({channels}) must be divisible by nheads ({nheads})")
        if window % 2 != 1:
            raise AssertionError(f"filter size M={window} must be odd.")
        self.window, self.nheads, self.simfun = window, nheads, simfun
        self.eps, self.fused = eps, fused
        self.theta = torch.nn.Linear(feat_channels, channels, bias=False)
        self.tau = torch.nn.Parameter(torch.full((channels,), float(tau)))

    def _theta(self, f: torch.Tensor) -> torch.Tensor:
        return self.theta(f)

    def adjacency(self, f: torch.Tensor) -> Circulant:
        """Γ (Julia size (P, P, nheads, B)) from features f (B, *spatial, F)."""
        th = self._theta(f).movedim(-1, 1).contiguous()  # planar (B, M, *spatial)
        return circulant_mh_adjacency(self.simfun, th, th, self.window, self.nheads)

    def energy(self, z: torch.Tensor, f: torch.Tensor = None, A: Circulant = None) -> torch.Tensor:
        """ξ = Γ ⨷ z² (channels-last, like z)."""
        z2 = z * z
        if A is not None:
            return Otimes(A, z2.movedim(-1, 1).contiguous()).movedim(1, -1).contiguous()
        if self.fused:
            dh = z.shape[-1] // self.nheads
            th = self._theta(f) * dh ** 0.25
            xi, _ = circulant_mh_attention(self.simfun, th, th, z2, self.window, self.nheads,
                                           materialize=False, honor_simfun=True,
                                           channels_last=True)
            return xi
        return self.energy(z, A=self.adjacency(f))

    def forward(self, z: torch.Tensor, f: torch.Tensor = None, A: Circulant = None) -> torch.Tensor:
        if f is None and A is None:
            raise AssertionError("GroupThresholding needs features f or an adjacency A")
        xi = self.energy(z, f, A)
        return z * torch.relu(1.0 - self.tau / torch.sqrt(xi + self.eps))


__all__ = ["CircAttBlock", "GroupThresholding", "SlidingAttBlock"]
