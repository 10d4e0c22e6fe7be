"""How the keys' gradients of sliding_mh_attention split their work (walk_split in
sliding.hip), restated, so that tests can pick shapes of each plan.  The
workspace that the library asks for follows from the plan, which pins the
restatement."""
import torch


def walk_split(B, L, H, Hk, D, W, S, dtype):
    """(parts of a block of 128 keys, groups of 32 sinks seen from behind their
    block's window, workgroups of each group, bytes of the workspace)."""
    G, units, blocks = H // Hk, B * Hk, (L + 127) // 128
    W, S = (L, 0) if W is None or W >= L else (W, min(S, L))
    rows = 32 if dtype == torch.float32 else 64
    DP = (D + 31) // 32 * 32
    walks = [min(L - 128 * k, 127 + W) * G / rows for k in range(blocks)]
    mean, longest, best, parts = sum(walks) / blocks, walks[0], float("inf"), 0
    for p in range(1, 9):
        rounds = (units * blocks * p + 255) // 256
        cost = max(rounds * (mean / p), longest / p) + rounds * (6 if p > 1 else 3)
        if cost < best:
            best, parts = cost, p
    far, far_parts, behind = 0, 1, L - 127 - W
    if S > 0 and behind > 0:
        far = (min(S, behind + 127) + 31) // 32
        most = 2048 // (units * far)
        far_parts = min((behind * G + 511) // 512, max(most, 1))
    floats = (B * L * H + 3) // 4 * 4 + units * far * far_parts * 64 * DP
    if parts > 1:
        floats += units * blocks * parts * 256 * DP
    return parts, far, far_parts, 4 * floats
