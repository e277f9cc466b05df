"""Attention of trees with one node's key or value spoilt: what every row is then, against the 64-bit oracle.

The nodes' keys weigh as much as the whole context here, so that a row that saw one ancestor too few or a node too many
would be several bars off (which `test_the_bars_tell_a_wrong_way` shows of the oracle, on the CPU)."""

from __future__ import annotations

import pytest
import torch

from oracle import tree_ref
from tests import tree_inputs

INF, NAN, LOWEST = float("inf"), float("nan"), torch.finfo(torch.bfloat16).min
CASES = [(8, 2, 64, 4, [40]), (16, 4, 128, 20, [100, 3]), (32, 2, 256, 16, [3000, 64]), (32, 2, 256, 2, [31]), (16, 4, 128, 40, [700])]


def bars(want, spread):
    """As in test_gpu_tree_attention: 2^-8 (spread + 2 |out|) for the rounded probabilities and output, 6e-4 of the spread for
    the fp32 scores behind them."""
    return 2.0**-8 * (spread + 2 * want.abs()) * (1 + 2.0**-7) + 6e-4 * spread + 1e-30


def case(heads, kvh, hd, t, base):
    """Positive queries, so that an infinite key's score is infinite and not NaN; small keys in the context, nodes whose
    weights add up to as much. Also the nodes' pool rows of lane 0, and the node to spoil, one with nodes below it where there are."""
    g = torch.Generator().manual_seed(t + hd)
    b, blocks = len(base), (max(base) + t + 15) // 16
    n = b * blocks + 1
    table = (torch.randperm(n - 1, generator=g) + 1).view(b, blocks).int()
    q = torch.randn(b, t, heads, hd, generator=g).abs().add(0.01).bfloat16()
    k, v = torch.randn(n * 16, kvh, hd, generator=g) * 0.5, torch.randn(n * 16, kvh, hd, generator=g)
    tree = tree_inputs.batch(["random"] * b, t, 1)
    tree[:, -1] = -2
    node_rows = []
    for j in range(b):
        pos = base[j] + torch.arange(t)
        rows = table[j].long()[pos // 16] * 16 + pos % 16
        # sum(q) is some 0.8 hd, so a key raised by x in every channel scores 0.8 sqrt(hd) x more
        k[rows] += torch.tensor(max(base[j] / max(t // 4, 1), 1.0)).log() / (0.8 * hd**0.5)
        node_rows.append(rows)
    spoilt = max(range(t - 1), key=lambda s: (sum(w is not None and s in w for w in tree_ref.ways(tree[0])) if s or t == 2 else 0))
    return q, k.bfloat16(), v.bfloat16(), table, torch.tensor(base), tree, node_rows[0], spoilt


def oracle(q, k, v, table, base, tree, hd):
    return tree_ref.attention(q, k, v, table, base, hd**-0.5, tree)


@pytest.mark.parametrize("heads,kvh,hd,t,base", CASES)
def test_the_bars_tell_a_wrong_way(heads, kvh, hd, t, base) -> None:
    """The oracle without one ancestor, or with one node more, is past the bars in the rows that this is about."""
    q, k, v, table, b0, tree, _, spoilt = case(heads, kvh, hd, t, base)
    want, spread = oracle(q, k, v, table, b0, tree, hd)
    ways = tree_ref.ways(tree[0])
    for s in [s for s, w in enumerate(ways) if w is not None and spoilt in w and s != spoilt][:3]:
        other = tree.clone()  # s hangs below the spoilt node's parent: its way without that node
        way = ways[s]
        for a in way[way.index(spoilt) + 1 :]:
            if int(tree[0, a]) == spoilt:
                other[0, a] = tree[0, spoilt]
        off, _ = oracle(q, k, v, table, b0, other, hd)
        assert float(((off - want).abs() / bars(want, spread))[0, s].max()) > 4.0
    clear = [s for s, w in enumerate(ways) if w is not None and spoilt not in w and s > spoilt]
    for s in clear[:3]:
        other = tree.clone()  # s with the spoilt node on its way
        other[0, s] = spoilt
        off, _ = oracle(q, k, v, table, b0, other, hd)
        assert float(((off - want).abs() / bars(want, spread))[0, s].max()) > 4.0


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kvh,hd,t,base", CASES)
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("worst", [NAN, INF, -INF, LOWEST])
def test_rows_with_a_spoilt_node(dev, heads, kvh, hd, t, base, what, worst) -> None:
    """Finite rows are the oracle's within its bars, and infinite and NaN channels are where the oracle has them: a key of
    minus infinity (or whose score is past fp32's range) weighs nothing, one of infinity leaves its rows NaN, and an infinite
    value makes infinite what sees it."""
    from tests.test_gpu_tree_attention import run

    q, k, v, table, b0, tree, rows, spoilt = case(heads, kvh, hd, t, base)
    (k if what == "k" else v)[rows[spoilt]] = worst
    want, spread = oracle(q, k, v, table, b0, tree, hd)
    below = torch.tensor([w is not None and spoilt in w for w in tree_ref.ways(tree[0])])
    assert bool(below.any()) and bool(want[0, ~below].isfinite().all()) and bool(want[1:].isfinite().all())
    got = run(dev, q, k, v, table, b0, hd**-0.5, tree).double().cpu()
    finite = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    assert float(((got - want).abs() / bars(want, spread))[finite].max()) <= 1.0
    assert not got[:, -1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kvh,hd,t,base", CASES)
def test_rows_beside_spoilt_memory(dev, heads, kvh, hd, t, base) -> None:
    """Every pool row that no present node is at, and none of the context's, is NaN, and so is the query of an absent node."""
    from tests.test_gpu_tree_attention import run

    q, k, v, table, b0, tree, _, _ = case(heads, kvh, hd, t, base)
    want, spread = oracle(q, k, v, table, b0, tree, hd)
    used = torch.zeros(k.shape[0], dtype=torch.bool)
    for j in range(len(base)):
        pos = torch.arange(base[j] + t - 1)
        used[table[j].long()[pos // 16] * 16 + pos % 16] = True
    k[~used], v[~used], q[:, -1] = NAN, NAN, NAN
    got = run(dev, q, k, v, table, b0, hd**-0.5, tree).double().cpu()
    assert not got[:, -1].any()
    assert float(((got - want).abs() / bars(want, spread)).max()) <= 1.0
