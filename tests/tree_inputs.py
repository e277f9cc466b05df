"""Trees for the tests: parents `[t]` of named shapes."""

from __future__ import annotations

import torch

SHAPES = ("chain", "star", "forest", "random", "deep", "gaps", "empty", "absent_root")


def parents(kind: str, t: int, seed: int = 0) -> list[int]:
    g = torch.Generator().manual_seed(1000 * t + seed)
    if kind == "chain":
        return list(range(-1, t - 1))
    if kind == "star":
        return [-1] + [0] * (t - 1)
    if kind == "forest":  # several nodes below the context itself
        return [-1 if s % 3 == 0 else s - 1 - int(torch.randint(0, s % 3, (1,), generator=g)) for s in range(t)]
    if kind == "random":
        return [-1] + [int(torch.randint(0, s, (1,), generator=g)) for s in range(1, t)]
    if kind == "deep":  # two chains that take turns
        return [-1] + [max(s - 2, 0) for s in range(1, t)]
    if kind == "gaps":  # a smaller tree's end, an absent node inside with nodes below it, values that are no parent
        p = parents("random", t, seed)
        for s in range(t):
            if s % 5 == 3:
                p[s] = [-2, s, s + 1, -(2**31), 2**31 - 1][s // 5 % 5]
        return p[: t - t // 4] + [-2] * (t // 4)
    if kind == "empty":
        return [-2] * t
    if kind == "absent_root":
        return [-2] + [s - 1 for s in range(1, t)]
    raise ValueError(kind)


def batch(kinds, t: int, seed: int = 0, dtype: torch.dtype = torch.int32) -> torch.Tensor:
    return torch.tensor([parents(kind, t, seed + j) for j, kind in enumerate(kinds)], dtype=dtype)
