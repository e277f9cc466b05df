"""Acceptance of a path and the move of its cache rows on the device, entry by entry against the oracle."""

from __future__ import annotations

import pytest
import torch

import attention
import graph_mtp
from oracle import tree_ref
from tests import tree_inputs

pytestmark = pytest.mark.gpu


def accept_case(b, t, seed, words=3):
    g = torch.Generator().manual_seed(seed)
    best, tokens = (torch.randint(0, words, (b, t), generator=g) for _ in range(2))
    kinds = [tree_inputs.SHAPES[int(torch.randint(0, len(tree_inputs.SHAPES), (1,), generator=g))] for _ in range(b)]
    tree = tree_inputs.batch(kinds, t, seed)
    up = tree.long().clamp(0, t - 1)
    follow = torch.rand(b, t, generator=g) < 0.6  # most nodes are what their parent's model says
    tokens = torch.where(follow, best.gather(1, up), tokens)
    stops = torch.full((b, 5), -1)
    stops[::3, 1] = words - 1
    return (best, tokens, tree, torch.rand(b, generator=g) < 0.8, torch.randint(0, 10**12, (b,), generator=g),
            torch.randint(-1, 9, (b,), generator=g), stops)


def same(got, want) -> None:
    for name, value in want.items():
        x = getattr(got, name).cpu()
        assert x.dtype == (torch.bool if name in ("keep", "live") else torch.int64)
        assert x.tolist() == value, name


@pytest.mark.parametrize("b,t", [(1, 1), (1, 7), (5, 2), (40, 16), (70, 33), (9, 64), (1500, 12)])
def test_acceptance(dev, b, t) -> None:
    args = accept_case(b, t, b + t)
    want = tree_ref.accept(*(x.tolist() for x in args))
    same(graph_mtp.tree_accept(*(x.to(dev) for x in args)), want)
    best, tokens, tree, *rest = args
    # strides: columns of wider buffers, a 64-bit tree
    wide = torch.zeros(b, t + 3, dtype=torch.long)
    wide[:, :t] = best
    same(graph_mtp.tree_accept(wide.to(dev)[:, :t], tokens.t().contiguous().to(dev).t(), tree.long().to(dev), *(x.to(dev) for x in rest)),
         want)


def test_acceptance_of_a_chain(dev) -> None:
    best, tokens, _, active, pos, budget, stops = (x.to(dev) for x in accept_case(64, 5, 3))
    tokens[:, 1:] = torch.where(torch.rand(64, 4, device=dev) < 0.7, best[:, :-1], tokens[:, 1:])
    got = graph_mtp.tree_accept(best, tokens, tree_inputs.batch(["chain"] * 64, 5).to(dev), active, pos, budget, stops)
    want = graph_mtp.greedy_accept(best, tokens[:, 1:], active, pos, budget, stops, 3)
    for name in ("accept_len", "lengths", "keep", "bonus", "next_pos", "budget_left", "live", "hidden_src"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name


def test_acceptance_without_stops_and_empty(dev) -> None:
    args = list(accept_case(6, 9, 1))
    args[-1] = torch.empty(6, 0, dtype=torch.long)
    same(graph_mtp.tree_accept(*(x.to(dev) for x in args)), tree_ref.accept(*(x.tolist() for x in args)))
    none = graph_mtp.tree_accept(*(x[:0].to(dev) for x in args))
    assert none.path.shape == (0, 9) and none.live.shape == (0,)


def keep_case(layers, b, t, kvh, hd, base, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + t)
    blocks = (max(base) + t + 15) // 16
    n = b * blocks + 2
    table = (torch.randperm(n - 1, generator=g)[: b * blocks] + 1).view(b, blocks).int()
    rows = [torch.randn(n * 16, kvh, hd, generator=g).to(dtype) for _ in range(2 * layers)]
    lengths = torch.tensor([min(1 + 5 * j % max(t, 1), t) if j else t for j in range(b)])
    path = torch.zeros(b, t, dtype=torch.long)
    for j in range(b):
        m = int(lengths[j])
        some = torch.cat([torch.tensor([0]), 1 + torch.randperm(t - 1, generator=g)[: m - 1]]).sort().values
        path[j] = torch.cat([some, some[-1:].expand(t - m)])
    return rows, table, torch.tensor(base), path, lengths


def pools_of(rows, dev):
    half = len(rows) // 2
    return [x.clone().to(dev) for x in rows[:half]] + [attention.v_blocks(x).to(dev) for x in rows[half:]]


def rows_of(pools):
    return [p.cpu() if p.dim() == 3 else attention.v_rows(p).cpu() for p in pools]


@pytest.mark.parametrize("layers,b,t,kvh,hd,base,dtype", [
    (1, 1, 2, 1, 8, [14], torch.bfloat16), (15, 3, 7, 2, 256, [299, 0, 16], torch.bfloat16), (2, 4, 61, 4, 128, [5, 31, 100, 48], torch.bfloat16),
    (40, 2, 16, 1, 24, [9, 15], torch.float32), (1, 2, 64, 5, 256, [7, 33], torch.float16), (1, 2, 33, 3, 100, [0, 1], torch.float32),
    (2, 3, 1, 2, 64, [4, 5, 6], torch.bfloat16), (3, 60, 9, 2, 64, list(range(60)), torch.bfloat16),
])  # fmt: skip
def test_kept_rows(dev, layers, b, t, kvh, hd, base, dtype) -> None:
    rows, table, b0, path, lengths = keep_case(layers, b, t, kvh, hd, base, dtype)
    pools = pools_of(rows, dev)
    want = [tree_ref.keep_rows(x, table.tolist(), base, path.tolist(), lengths.tolist()) for x in rows]
    attention.keep_path(pools, table.to(dev), b0.to(dev), path.to(dev), lengths.to(dev))
    assert all(torch.equal(x, y) for x, y in zip(rows_of(pools), want))
    cpu = pools_of(rows, "cpu")
    attention.keep_path(cpu, table, b0, path, lengths)
    assert all(torch.equal(x, y) for x, y in zip(rows_of(cpu), want))


def test_kept_rows_that_lie_outside(dev) -> None:
    """Entries that are no node end a path; blocks outside the pools and positions outside the table are left; lengths past
    the nodes are all of them."""
    rows, table, b0, path, lengths = keep_case(1, 4, 12, 2, 64, [20, 3, 40, 60], torch.bfloat16)
    table = torch.cat([table, torch.zeros(4, 1, dtype=torch.int32)], 1)
    path[:] = torch.arange(12).div(2, rounding_mode="floor") + torch.arange(12)  # 0 1 3 4 6 7 9 10, then past the nodes
    lengths = torch.tensor([2**40, 12, -3, 12])
    table[1, 1], b0[3] = -7, 5000
    pools, cpu = pools_of(rows, dev), pools_of(rows, "cpu")
    attention.keep_path(pools, table.to(dev), b0.to(dev), path.int().to(dev), lengths.to(dev))
    attention.keep_path(cpu, table, b0, path, lengths)
    got, want = rows_of(pools), rows_of(cpu)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    first = tree_ref.keep_rows(rows[0], table.tolist(), [20], [path[0, :8].tolist()], [8])
    lane = torch.arange(48)
    at = table[0].long()[lane // 16] * 16 + lane % 16
    assert torch.equal(got[0][at], first[at])
    at = table[2].long()[lane // 16] * 16 + lane % 16
    assert torch.equal(got[0][at], rows[0][at])


def test_in_a_graph(dev) -> None:
    args = [x.to(dev) for x in accept_case(6, 20, 7, words=2)]
    rows, table, b0, _, _ = keep_case(2, 6, 20, 2, 64, [3, 20, 40, 7, 15, 16], torch.bfloat16)
    table, b0 = table.to(dev), b0.to(dev)

    def step(pools):
        r = graph_mtp.tree_accept(*args)
        attention.keep_path(pools, table, b0, r.path, r.lengths)
        return r

    mine, eager = pools_of(rows, dev), pools_of(rows, dev)
    step(pools_of(rows, dev))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(mine)
    for i in range(4):
        for x, y in zip(args, accept_case(6, 20, 50 + i, words=2)):
            x.copy_(y)
        graph.replay()
        want = step(eager)
        assert all(torch.equal(getattr(got, n), getattr(want, n)) for n in got.__dataclass_fields__)
        assert all(torch.equal(x, y) for x, y in zip(mine, eager))


def test_pools_that_share_memory_are_refused(dev) -> None:
    rows, table, b0, path, lengths = keep_case(1, 2, 8, 2, 64, [3, 9], torch.bfloat16)
    k, v = pools_of(rows, dev)
    args = (table.to(dev), b0.to(dev), path.to(dev), lengths.to(dev))
    for pools in ([k, v, k], [k, k.view(-1, 2, 64, 16)]):
        with pytest.raises(ValueError, match="no two of one memory"):
            attention.keep_path(pools, *args)
    assert torch.equal(k.cpu(), rows[0])


def test_the_lowest_budget_accepts_nothing(dev) -> None:
    best, tokens, tree, active, pos, budget, stops = (x.to(dev) for x in accept_case(5, 9, 2, words=1))
    budget[:] = -(2**63) + 70
    got = graph_mtp.tree_accept(best, tokens, tree, active, pos, budget, stops)
    assert got.accept_len.tolist() == [0] * 5 and not got.live.any()
