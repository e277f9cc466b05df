"""The trees' oracle on chains, where it has to be the chain's, and what must not matter to a node."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import accept_ref, attention_ref, deltanet_ref, tree_ref
from tests import tree_inputs


def _rule(seed, b=2, t=5, heads=2, dk=16, dv=8):
    r = np.random.default_rng(seed)
    state = r.standard_normal((3, heads, dk, dv))
    q, k = (r.standard_normal((b, t, 1, dk)) / 4 for _ in range(2))
    return state, [2, 0], q, k, r.standard_normal((b, t, heads, dv)), -r.random((b, t, heads)), r.random((b, t, heads))


def test_ways() -> None:
    assert tree_ref.ways([-1, 0, 0, 1, -2, 4, 2]) == [[0], [0, 1], [0, 2], [0, 1, 3], None, None, [0, 2, 6]]
    assert tree_ref.ways([0, -1, 5]) == [None, [1], None]


def test_rule_on_a_chain_and_along_ways() -> None:
    args = _rule(0)
    chain = tree_inputs.batch(["chain", "chain"], 5)
    np.testing.assert_allclose(tree_ref.delta_rule(*args, chain), deltanet_ref.delta_rule_rows(*args)[1], rtol=1e-13)
    tree = tree_inputs.batch(["random", "gaps"], 5)
    got = tree_ref.delta_rule(*args, tree)
    state, slots, *rows = args
    for j in range(2):
        for s, way in enumerate(tree_ref.ways(tree[j])):
            if way is None:
                assert not got[j, s].any()
            else:
                want = deltanet_ref.delta_rule_rows(state, slots[j : j + 1], *(x[j : j + 1, way] for x in rows))[1]
                np.testing.assert_allclose(got[j, s], want[0, -1], rtol=1e-13)


def test_commit_on_a_prefix() -> None:
    state, slots, q, k, v, g, beta = _rule(1)
    raw, conv = np.random.default_rng(3).standard_normal((2, 5, 6)), np.random.default_rng(4).standard_normal((3, 6, 3))
    path, lengths = np.tile(np.arange(5), (2, 1)), [4, 0]
    got, win = tree_ref.commit(state, conv, slots, k, v, g, beta, path, lengths, raw)
    np.testing.assert_allclose(got, deltanet_ref.delta_rule_rows(state, slots, q, k, v, g, beta, lengths)[0], rtol=1e-13)
    np.testing.assert_array_equal(win[2], raw[0, 1:4].T)
    np.testing.assert_array_equal(win[:2], conv[:2])


def test_convolution() -> None:
    r = np.random.default_rng(5)
    conv, w, raw = r.standard_normal((2, 4, 3)), r.standard_normal((4, 4)), r.standard_normal((1, 6, 4))
    got = tree_ref.conv_rows(conv, [1], w, raw, [[-1, 0, 1, 0, 3, -2]])
    line = np.concatenate([conv[1], raw[0].T], axis=1)
    for s in range(3):  # the first three nodes are a chain
        np.testing.assert_allclose(got[0, s], (line[:, s : s + 4] * w).sum(1))
    other = np.concatenate([conv[1], raw[0, [0, 3, 4]].T], axis=1)
    np.testing.assert_allclose(got[0, 4], (other[:, 2:6] * w).sum(1))
    assert not got[0, 5].any()


def test_attention_on_a_chain_and_off_the_way() -> None:
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(*s, generator=g) for s in ((2, 5, 4, 8), (96, 2, 8), (96, 2, 8)))
    table, base = torch.tensor([[3, 1, 0], [5, 2, 4]]), torch.tensor([14, 0])
    chain = tree_inputs.batch(["chain", "chain"], 5)
    got, _ = tree_ref.attention(q, k, v, table, base, 0.3, chain)
    want = attention_ref.paged_attention(q.transpose(1, 2).numpy(), k.numpy(), v.numpy(), table.numpy(), base.numpy(), 0.3)
    np.testing.assert_allclose(got.transpose(1, 2).numpy(), want, rtol=1e-12)
    tree = tree_inputs.batch(["star", "star"], 5)
    one, _ = tree_ref.attention(q, k, v, table, base, 0.3, tree)
    v[3 * 16 + 15] = 100.0  # node 1 of lane 0
    two, _ = tree_ref.attention(q, k, v, table, base, 0.3, tree)
    assert torch.equal(one[:, [0, 2, 3, 4]], two[:, [0, 2, 3, 4]]) and not torch.equal(one[0, 1], two[0, 1])


@pytest.mark.parametrize("seed", range(4))
def test_acceptance_of_a_chain(seed) -> None:
    r = np.random.default_rng(seed)
    b, t = 16, 6
    best, tokens = r.integers(0, 3, (b, t)), r.integers(0, 3, (b, t))
    tokens[:, 1:] = np.where(r.random((b, t - 1)) < 0.8, best[:, :-1], tokens[:, 1:])
    stops = np.full((b, 3), -1)
    stops[::4, 0] = 2
    budget, pos, active = r.integers(0, 8, b), r.integers(0, 90, b), r.random(b) < 0.7
    got = tree_ref.accept(best.tolist(), tokens.tolist(), [list(range(-1, t - 1))] * b, active.tolist(), pos.tolist(), budget.tolist(),
                          stops.tolist())
    for j in range(b):
        n = accept_ref.commit_limit(accept_ref.greedy_accept_length(tokens[j, 1:], best[j, :-1]), best[j].tolist(), int(budget[j]),
                                    set(stops[j].tolist()) - {-1})
        assert got["accept_len"][j] == n and got["path"][j] == list(range(n + 1)) + [n] * (t - n - 1)
        assert got["bonus"][j] == best[j, n] and got["lengths"][j] == (n + 1 if active[j] else 1)


def test_kept_rows() -> None:
    rows = torch.arange(64.0)[:, None]
    same = tree_ref.keep_rows(rows, [[2, 1]], [3], [[0, 1, 2, 2]], [3])
    assert torch.equal(same, rows)
    moved = tree_ref.keep_rows(rows, [[2, 1]], [14], [[0, 2, 3]], [3])
    assert moved[47, 0] == 16 and moved[16, 0] == 17 and moved[46, 0] == 46
