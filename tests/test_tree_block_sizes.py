"""A round over trees in caches whose blocks are not of 16 rows."""

from __future__ import annotations

import dataclasses

import pytest
import torch

import attention
import mtp
import verify_model as vm
from oracle import tree_ref
from tests import model_helpers as mh
from tests import tree_inputs, tree_round


def build(block: int, device: str = "cpu") -> vm.Model:
    model = vm.Model(dataclasses.replace(vm.tiny_cfg(), block_size=block), device, torch.float32, lanes=2, max_seq=96, seed=0)
    mtp.attach(model, k=1, seed=1)
    return model


# Rows of a tree and of plain decode sum their products in different orders. A sum of 64 products is off by at most 64 x 2^-24
# of its terms' magnitudes, which add up to some 64 x 0.64 against a result of sqrt(64): 64 x 2^-24 x 5.1 = 2e-5 of a result of 1.
# A cached row of 1 in the square mean lies behind five such sums or more (in and out projection, the expert's two, its own): 1e-4.
TOL = 1e-4


def rounds(model: vm.Model, seq: vm.Model) -> None:
    ids = mh.prompts()
    truth = mh.greedy_truth(build(model.cfg.block_size), ids, 30)
    for lane, p in enumerate(ids):
        model.prefill(lane, p), seq.prefill(lane, p)
    at = [0, 0]
    for rnd in range(3):
        trees = [tree_round.planted("random", 9, truth[j][at[j] :], model.cfg.vocab, 10 * rnd + j) for j in range(2)]
        tokens, parents = [x[0] for x in trees], [x[1] for x in trees]
        out = tree_round.run(model, [0, 1], tokens, parents, [16 + a for a in at], 64)
        for j in range(2):
            got = tree_round.committed(out, tokens, j)
            assert len(got) > trees[j][2] and got == truth[j][at[j] + 1 : at[j] + 1 + len(got)]
            at[j] += len(got)
    for lane in range(2):
        vm.greedy_reference(seq, lane, truth[lane][0], 16, at[lane])
        mh.assert_slot_state_close(model, seq, lane, 16 + at[lane], rtol=TOL, atol=TOL)


@pytest.mark.parametrize("block", [4, 32])
def test_rounds_match_greedy(block) -> None:
    rounds(build(block), build(block))


def kept(device, block: int, t: int = 11):
    """(pools, what they hold after, the call's other operands)."""
    g = torch.Generator().manual_seed(block)
    base, lengths = torch.tensor([13, 30, 5]), torch.tensor([t, 5, 3])
    per = (30 + t + block - 1) // block
    table = (torch.randperm(3 * per, generator=g) + 1).view(3, per).int()
    rows = [torch.randn((3 * per + 1) * block, 2, 8, generator=g) for _ in range(2)]
    path = torch.stack([torch.cat([torch.zeros(1).long(), (1 + torch.randperm(t - 1, generator=g)[: int(n) - 1]).sort().values,
                                   torch.full((t - int(n),), t)]) for n in lengths])  # t is no node
    want = [tree_ref.keep_rows(x, table.tolist(), base.tolist(), path.tolist(), lengths.tolist(), block) for x in rows]
    pools = [rows[0].to(device), attention.v_blocks(rows[1], block).to(device)]
    return pools, want, [x.to(device) for x in (table, base, path, lengths)]


def same(pools, want) -> bool:
    return torch.equal(pools[0].cpu(), want[0]) and torch.equal(attention.v_rows(pools[1]).cpu(), want[1])


@pytest.mark.parametrize("block", [1, 4, 16, 48])
def test_kept_rows(block) -> None:
    pools, want, args = kept("cpu", block)
    attention.keep_path(pools, *args, block)
    assert same(pools, want)


def test_nothing_to_keep() -> None:
    pools, _, (table, base, path, lengths) = kept("cpu", 4)
    before = [p.clone() for p in pools]
    attention.keep_path(pools, table, base, path, torch.zeros_like(lengths), 4)
    attention.keep_path(pools, torch.full_like(table, -1), base, path, lengths, 4)
    attention.keep_path(pools, table[:0], base[:0], path[:0], lengths[:0], 4)
    assert all(torch.equal(x, y) for x, y in zip(pools, before))


def test_a_block_size_that_does_not_fit_is_refused() -> None:
    pools, _, args = kept("cpu", 4)
    for block in (16, 3, 0):
        with pytest.raises(ValueError):
            attention.keep_path(pools, *args, block)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 4, 16, 48])
def test_kept_rows_on_the_device_and_in_a_graph(dev, block) -> None:
    pools, want, args = kept(dev, block)
    first = [p.clone() for p in pools]
    attention.keep_path(pools, *args, block)
    assert same(pools, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention.keep_path(pools, *args, block)
    for _ in range(3):
        for p, x in zip(pools, first):
            p.copy_(x)
        graph.replay()
        assert same(pools, want)


@pytest.mark.gpu
def test_rounds_match_greedy_on_the_device(dev) -> None:
    rounds(build(4, dev), build(4, dev))
