"""Trees of drafts on the CPU: their masks, depths and acceptance against the oracle, the model's rounds against greedy decode,
and the refusals that need no device."""

from __future__ import annotations

import pytest
import torch

import attention
import deltanet
import graph_mtp
import verify_model as vm
from oracle import tree_ref
from tests import model_helpers as mh
from tests import tree_inputs, tree_round


@pytest.mark.parametrize("t", [1, 2, 3, 7, 16, 33, 64])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_ancestors_and_depths(t, dtype) -> None:
    tree = tree_inputs.batch(tree_inputs.SHAPES, t, 3, dtype)
    above, depths = vm.tree_ancestors(tree), vm.tree_depths(tree)
    for j, p in enumerate(tree.tolist()):
        for s, way in enumerate(tree_ref.ways(p)):
            assert above[j, s].nonzero()[:, 0].tolist() == (way or [])
            assert int(depths[j, s]) == (len(way) - 1 if way else 0)


def test_depths_of_values_past_32_bits() -> None:
    tree = torch.tensor([[-1, 0, 2**32, 1, -(2**63)]])
    assert vm.tree_depths(tree).tolist() == [[0, 1, 0, 2, 0]]
    assert vm.tree_ancestors(tree)[0, 2].any().item() is False


@pytest.mark.parametrize("b,t", [(1, 1), (9, 6), (20, 33), (3, 64)])
def test_acceptance(b, t) -> None:
    g = torch.Generator().manual_seed(t)
    tree = tree_inputs.batch([tree_inputs.SHAPES[j % len(tree_inputs.SHAPES)] for j in range(b)], t, 1)
    best, tokens = (torch.randint(0, 3, (b, t), generator=g) for _ in range(2))
    stops = torch.full((b, 3), -1)
    stops[::2, 1] = 2
    args = (best, tokens, tree, torch.rand(b, generator=g) < 0.7, torch.arange(b), torch.randint(-1, 6, (b,), generator=g), stops)
    want = tree_ref.accept(*(x.tolist() for x in args))
    got = graph_mtp.tree_accept(*args)
    for name, value in want.items():
        assert getattr(got, name).tolist() == value, name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kept_rows(dtype) -> None:
    g = torch.Generator().manual_seed(2)
    table = torch.tensor([[5, 2, 7], [1, 6, 3]], dtype=torch.int32)
    rows = [torch.randn(8 * 16, 2, 8, generator=g).to(dtype) for _ in range(2)]
    path = torch.tensor([[0, 2, 3, 9, 9, 9, 9, 9, 9, 9], [0, 1, 5, 6, 7, 7, 7, 7, 7, 7]])
    base, lengths = torch.tensor([13, 30]), torch.tensor([4, 5])
    want = [tree_ref.keep_rows(x, table.tolist(), base.tolist(), path.tolist(), lengths.tolist()) for x in rows]
    pools = [rows[0].clone(), attention.v_blocks(rows[1])]
    attention.keep_path(pools, table, base, path, lengths)
    assert torch.equal(pools[0], want[0]) and torch.equal(attention.v_rows(pools[1]), want[1])


def test_a_chain_is_the_rows_forward() -> None:
    ids = mh.prompts()
    a, b = mh.build(), mh.build()
    for lane, p in enumerate(ids):
        a.prefill(lane, p), b.prefill(lane, p)
    tokens = torch.tensor(mh.prompts(2, 5, seed=9))
    pos = torch.tensor([16, 16])
    for m in (a, b):
        m.blocks.grow_many([0, 1], [21, 21])
    want = a.forward_rows(tokens, [0, 1], pos, 21)
    got = b.forward_rows(tokens, [0, 1], pos, 21, parents=tree_inputs.batch(["chain"] * 2, 5))
    torch.testing.assert_close(got.hidden, want.hidden, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("kind", ["chain", "star", "random", "deep"])
@pytest.mark.parametrize("t", [1, 4, 16])
def test_rounds_match_greedy(kind, t) -> None:
    """Trees round after round commit what plain decode commits, and leave the slots where it leaves them."""
    ids, steps = mh.prompts(), 24
    truth = mh.greedy_truth(mh.build(), ids, steps + 20)
    model, seq = mh.build(), mh.build()
    pos, at = [len(p) for p in ids], [0, 0]
    for m in (model, seq):
        for lane, p in enumerate(ids):
            m.prefill(lane, p)
    rnd = 0
    while min(at) < steps:
        lanes = [0, 1] if at[0] < steps and at[1] < steps else [0 if at[0] < steps else 1]
        trees = [tree_round.planted(kind, t, truth[j][at[j] : steps + 1], model.cfg.vocab, 10 * rnd + j) for j in lanes]
        tokens, parents = [x[0] for x in trees], [x[1] for x in trees]
        left = [steps - at[j] for j in lanes]
        out = tree_round.run(model, lanes, tokens, parents, [pos[j] + at[j] for j in lanes], 96, budget=left)
        for i, j in enumerate(lanes):
            got = tree_round.committed(out, tokens, i)
            assert len(got) >= min(trees[i][2] + 1, left[i])
            assert got == truth[j][at[j] + 1 : at[j] + 1 + len(got)]
            at[j] += len(got)
        rnd += 1
    for lane, p in enumerate(ids):
        vm.greedy_reference(seq, lane, truth[lane][0], pos[lane], at[lane])
        mh.assert_slot_state_close(model, seq, lane, pos[lane] + at[lane])


def test_inactive_rows_touch_nothing() -> None:
    model = mh.build()
    for lane, p in enumerate(mh.prompts()):
        model.prefill(lane, p)
    model.blocks.grow_many([0, 1], [21, 21])
    before = mh.slot_state(model, 1, 16)
    trees = [tree_inputs.parents("random", 5, s) for s in range(2)]
    tree_round.run(model, [0, 1], mh.prompts(2, 5, seed=1), trees, [16, 16], 21, active=[True, False])
    assert all(torch.equal(x, y) for x, y in zip(before, mh.slot_state(model, 1, 16), strict=True))


@pytest.mark.parametrize("pad,like", [(-100, 0), (2**40, vm.tiny_cfg().vocab - 1)])
def test_padded_trees_may_hold_any_ids(pad, like) -> None:
    """Trees of different sizes in one batch: absent nodes and an inactive lane may hold ids that are no ids. They count as the
    nearest id, so the batch is the same to the last bit (another id there changes which rows an expert's product sums together)."""
    outs, states = [], []
    for fill in (pad, like):
        model = mh.build(lanes=3)
        for lane, p in enumerate(mh.prompts(3)):
            model.prefill(lane, p)
        tokens = mh.prompts(3, 6, seed=4)
        tokens[0][4:], tokens[2][:] = [fill] * 2, [fill] * 6
        parents = [[-1, 0, 0, 1, -2, 4], [-1, 0, 1, 1, 0, 4], [-1, 0, 1, 2, 3, 4]]
        out = tree_round.run(model, [0, 1, 2], tokens, parents, [16] * 3, 22, active=[True, True, False])
        outs.append([out.path[:2], out.accept_len[:2], out.bonus[:2]])
        states.append([x for j in range(3) for x in mh.slot_state(model, j, 16 + (int(out.lengths[j]) if j < 2 else 0))])
    for x, y in zip(outs[0] + states[0], outs[1] + states[1], strict=True):
        assert torch.equal(x, y)


def test_a_budget_of_the_lowest_value_accepts_nothing() -> None:
    b = torch.tensor([[1, 2]])
    got = graph_mtp.tree_accept(b, torch.tensor([[0, 1]]), torch.tensor([[-1, 0]]), torch.tensor([True]), torch.tensor([3]),
                                torch.tensor([-(2**63) + 9]), torch.full((1, 1), -1))
    assert got.accept_len.tolist() == [0] and got.live.tolist() == [False]


def test_the_model_refuses_trees_of_other_sizes() -> None:
    model = mh.build()
    with pytest.raises(ValueError, match="parents must be"):
        model.forward_rows(torch.zeros(1, 4, dtype=torch.long), [0], torch.tensor([0]), 4, parents=torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="1 to 64 nodes"):
        model.forward_rows(torch.zeros(1, 65, dtype=torch.long), [0], torch.tensor([0]), 65, parents=torch.zeros(1, 65, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32 or int64"):
        model.forward_rows(torch.zeros(1, 2, dtype=torch.long), [0], torch.tensor([0]), 2, parents=torch.zeros(1, 2))


def test_kept_rows_refusals() -> None:
    k = torch.zeros(32, 2, 8)
    table, base = torch.ones(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.long)
    path, n = torch.zeros(1, 4, dtype=torch.long), torch.ones(1, dtype=torch.long)
    for bad in (([], table, base, path, n), ([k], table, base, path[0], n), ([k], table, base, torch.zeros(1, 65, dtype=torch.long), n),
                ([k], table, base, path.float(), n), ([k], table, base, path, n.repeat(2)), ([k[:31]], table, base, path, n),
                ([k, torch.zeros(3, 2, 8, 16)], table, base, path, n), ([k, k], table, base, path, n),
                ([k, k.view(2, 2, 8, 16)], table, base, path, n)):
        with pytest.raises(ValueError):
            attention.keep_path(*bad)


def test_device_operators_refuse_cpu_tensors() -> None:
    q, k, v = torch.zeros(1, 2, 2, 64).bfloat16(), torch.zeros(32, 1, 64).bfloat16(), torch.zeros(2, 1, 64, 16).bfloat16()
    tree, base = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.long)
    with pytest.raises(ValueError):
        attention.paged_attention_tree(q, k, v, torch.ones(1, 1, dtype=torch.int32), base, 16, 0.1, tree)
    state, f = torch.zeros(1, 2, 64, 64), torch.zeros
    with pytest.raises(ValueError):
        deltanet.delta_rule_tree(state, base, f(1, 2, 1, 64), f(1, 2, 1, 64), f(1, 2, 2, 64), f(1, 2, 2), f(1, 2, 2), tree)
    with pytest.raises(ValueError):
        deltanet.prep_tree(f(1, 2, 260), f(1, 256, 3), base, f(256, 4), f(2), f(2), 1, 64, 2, 64, tree)
    with pytest.raises(ValueError):
        deltanet.commit_path(state, f(1, 256, 3), base, f(1, 2, 1, 64), f(1, 2, 2, 64), f(1, 2, 2), f(1, 2, 2), tree.long(), base,
                             f(1, 2, 260), 256)
