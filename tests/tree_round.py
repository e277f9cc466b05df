"""Rounds over trees for the model tests, on any device: a tree holds the greedy continuation on one of its ways."""

from __future__ import annotations

import torch

import graph_mtp
from tests import tree_inputs


def planted(kind: str, t: int, truth: list[int], vocab: int, seed: int) -> tuple[list[int], list[int], int]:
    """(tokens, parents, depth) of one lane: `truth[0]` at node 0, the following ids along one of the deepest ways below it, as
    far as `truth` lasts, everything else drawn at random."""
    g = torch.Generator().manual_seed(seed)
    parents = tree_inputs.parents(kind, t, seed)
    tokens = torch.randint(0, vocab, (t,), generator=g).tolist()
    ways: list[list[int] | None] = []
    for s, p in enumerate(parents):
        above = ways[p] if 0 <= p < s else None
        ways.append([0] if s == 0 else None if above is None else [*above, s])
    way = max((w for w in ways if w is not None), key=len)
    depth = min(len(way) - 1, len(truth) - 1)
    for i, s in enumerate(way[: depth + 1]):
        tokens[s] = truth[i]
    return tokens, parents, depth


def run(model, lanes, tokens, parents, pos, ctx_len, *, budget=None, stops=None, active=None) -> graph_mtp.TreeAccept:
    """`verify_tree` of host lists, with the lanes' blocks grown for every node."""
    dev, b, t = model.device, len(lanes), len(tokens[0])
    model.blocks.grow_many(lanes, [p + t for p in pos])
    on = lambda x, dtype=torch.int64: torch.tensor(x, dtype=dtype, device=dev)  # noqa: E731
    return graph_mtp.verify_tree(
        model, on(lanes), on(tokens), on(parents, torch.int32), on(pos), on([10**6] * b if budget is None else budget),
        torch.full((b, 2), -1, device=dev) if stops is None else on(stops), ctx_len,
        active=None if active is None else on(active, torch.bool))


def committed(out: graph_mtp.TreeAccept, tokens, lane: int) -> list[int]:
    n = int(out.accept_len[lane])
    return [tokens[lane][s] for s in out.path[lane, 1 : n + 1].tolist()] + [int(out.bonus[lane])]
