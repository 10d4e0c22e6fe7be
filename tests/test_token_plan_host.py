"""The restated plan of the keys' gradients against the library's workspaces."""
import random

import pytest
import torch

from token_plan import walk_split

CODES = {torch.float32: 0, torch.float16: 2, torch.bfloat16: 3}


def test_restated_plan_gives_the_workspace():
    from circulant_attention import _lib as L
    rng, seen = random.Random(5), set()
    for _ in range(400):
        Hk, G = rng.randint(1, 12), rng.randint(1, 6)
        B, n, D = rng.randint(1, 9), int(2 ** rng.uniform(0, 12)), 8 * rng.randint(1, 16)
        W, S = rng.choice([None, int(2 ** rng.uniform(0, 11))]), rng.choice([0, int(2 ** rng.uniform(0, 9))])
        dtype = rng.choice(list(CODES))
        parts, far, _, size = walk_split(B, n, G * Hk, Hk, D, W, S, dtype)
        assert L.lib.circatt_sliding_bwd_workspace_bytes(CODES[dtype], n, B, G * Hk, Hk, D, W or 1 << 30, S) == size
        seen.add((min(parts, 2), min(far, 3)))
    assert {(1, 0), (2, 0), (1, 1), (2, 1), (1, 3), (2, 3)} <= seen
