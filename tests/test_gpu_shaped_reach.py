"""A token that is NaN reaches, under shaped scores, exactly what the definition makes NaN of it:

  q of row t     y and dq of row t, dk and dv of the keys that it sees
  k of key t     y and dq of the rows that see it, dk and dv of all keys that those see
  v of key t     the channel of y of the rows that see it, their dq, dk of the keys that those see;
                 not dv, which is of weights and dy alone
  dy of row t    dq of row t, dk and the channel of dv of the keys that it sees; not y

in the heads that share the token's."""
import pytest
import torch

import shaped_model as M

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
H, HK, D, L = 4, 2, 64, 300


@pytest.fixture(scope="module")
def ca(cuda):
    import circulant_attention
    return circulant_attention


def kinds(name):
    """(shape, W, S, see) of a call on L tokens."""
    i, W, S, start, P = torch.arange(L), 70, 3, None, 0
    shape = {}
    if "cap" in name:
        shape["cap"] = 20.0
    if "slopes" in name:
        shape["slopes"] = torch.tensor([0.2, 0.1, 0.05, 0.02], device="cuda")
    if "places" in name:
        places = torch.cat([torch.arange(n) for n in (40, 1, 130, L - 171)])
        shape["places"] = places.int()[None].cuda()
        start = i - places
    if "prefix" in name:
        P = 90
        shape["prefix"] = torch.tensor([P], dtype=torch.int32, device="cuda")
    return shape, W, S, M.visible(i, L, W, S, start, P)


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("kind", ["cap", "slopes", "places", "prefix", "cap places", "cap prefix", "cap slopes"])
@pytest.mark.parametrize("what,t", [(w, t) for w in ("q", "k", "v", "dy") for t in (0, 85, 171, 260)])
def test_a_nan_reaches_what_sees_it(ca, dtype, kind, what, t):
    dt = DT[dtype]
    shape, W, S, see = kinds(kind)
    g = torch.Generator().manual_seed(t)
    x = {n: torch.randn((1, L, h * D), generator=g).to(dt) for n, h in (("q", H), ("k", HK), ("v", HK), ("dy", H))}
    head, ch = (3, 5) if what in ("q", "dy") else (1, 5)      # of queries; of keys: heads 2 and 3 of queries
    x[what][0, t, head * D + ch] = float("nan")
    leaves = [x[n].cuda().requires_grad_(True) for n in ("q", "k", "v")]
    y = ca.sliding_mh_attention(*leaves, W, H, kv_heads=HK, sinks=S, **shape)
    dq, dk, dv = torch.autograd.grad(y, leaves, x["dy"].cuda())
    rows = torch.zeros(L, dtype=torch.bool)                   # that the token reaches, and the keys that they see
    if what in ("q", "dy"):
        rows[t] = True
    else:
        rows = see[:, t]
    keys = see[rows].any(0)
    want = {n: torch.zeros((L, h, D), dtype=torch.bool) for n, h in (("y", H), ("dq", H), ("dk", HK), ("dv", HK))}
    heads = [3] if what in ("q", "dy") else [2, 3]
    for h in heads:
        want["dq"][rows, h] = True
        if what == "v":
            want["y"][rows, h, ch] = True
        elif what != "dy":
            want["y"][rows, h] = True
    want["dk"][keys, 1] = True
    if what == "dy":
        want["dv"][keys, 1, ch] = True
    elif what != "v":
        want["dv"][keys, 1] = True
    for n, got in (("y", y.detach()), ("dq", dq), ("dk", dk), ("dv", dv)):
        bad = ~torch.isfinite(got[0].cpu().float()).reshape(want[n].shape)
        assert torch.equal(bad, want[n]), (n, "missed" if (want[n] & ~bad).any() else "reached too much",
                                           (bad != want[n]).nonzero()[:4].tolist())
