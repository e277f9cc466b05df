"""Attention of trees of drafts against its 64-bit oracle.

Bars as in test_gpu_attention_masked: 2^-8 (spread + 2 |out|) for the rounded probabilities and output, 6e-4 of the
spread for the fp32 scores behind them."""

from __future__ import annotations

import random

import pytest
import torch

import attention
from oracle import masked_attention_ref, tree_ref
from tests import tree_inputs

pytestmark = pytest.mark.gpu


def bars(want, spread):
    return 2.0**-8 * (spread + 2 * want.abs()) * (1 + 2.0**-7) + 6e-4 * spread + 1e-30


def case(seed, b, t, heads, kvh, hd, base, *, spare=1):
    g = torch.Generator().manual_seed(seed)
    blocks = max((max(base) + t + 15) // 16 + spare, 1)
    n = b * blocks + 1
    table = (torch.randperm(n - 1, generator=g) + 1).view(b, blocks).int()
    q = torch.randn(b, t, heads, hd, generator=g).bfloat16()
    k, v = (torch.randn(n * 16, kvh, hd, generator=g).bfloat16() for _ in range(2))
    return q, k, v, table, torch.tensor(base)


def run(dev, q, k, v, table, base, scale, parents, ctx=None, gate=None):
    ctx = max(int(base.max()) + q.shape[1], 0) if ctx is None else ctx
    return attention.paged_attention_tree(q.to(dev), k.to(dev), attention.v_blocks(v).to(dev), table.to(dev), base.to(dev), ctx,
                                          scale, parents.to(dev), gate=None if gate is None else gate.to(dev))


def check(dev, q, k, v, table, base, scale, parents, **kw):
    got = run(dev, q, k, v, table, base, scale, parents, **kw).double().cpu()
    want, spread = tree_ref.attention(q, k, v, table, base, scale, parents, kw.get("gate"))
    assert not bool(got.isnan().any())
    assert float(((got - want).abs() / bars(want, spread)).max()) <= 1.0
    absent = torch.tensor([[w is None for w in tree_ref.ways(p)] for p in parents])
    assert not got[absent].any()
    return got


LAYOUTS = [(8, 2, 64), (32, 2, 256), (16, 4, 128), (6, 2, 128), (4, 4, 64), (5, 1, 64)]
SIZES = [  # nodes, context
    (1, [0]), (1, [299, 15, 16]), (2, [40, 95]), (3, [13]), (7, [299, 31]), (16, [600, 0, 48]), (17, [250]), (31, [3, 64]),
    (32, [1000]), (33, [0, 700]), (61, [15]), (64, [0, 130]),
]  # fmt: skip


@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("t,base", SIZES)
def test_against_the_oracle(dev, t, base, heads, kvh, hd) -> None:
    kinds = ["random", "gaps", "star", "deep", "forest", "chain"]
    start = (t + hd + heads) % len(kinds)
    tree = tree_inputs.batch([kinds[(start + j) % len(kinds)] for j in range(len(base))], t)
    check(dev, *case(t + hd, len(base), t, heads, kvh, hd, base), hd**-0.5, tree)


@pytest.mark.parametrize("kind", tree_inputs.SHAPES)
@pytest.mark.parametrize("heads,kvh,hd,t", [(8, 2, 64, 7), (32, 2, 256, 16), (16, 4, 128, 40)])
def test_shapes_of_trees(dev, kind, heads, kvh, hd, t) -> None:
    g = torch.Generator().manual_seed(t)
    gate = torch.randn(3, t, heads, hd, generator=g).bfloat16()
    tree = tree_inputs.batch([kind, "random", kind], t, dtype=torch.int64)
    check(dev, *case(9, 3, t, heads, kvh, hd, [29, 500, 0]), hd**-0.5, tree, gate=gate)


def test_key_splits(dev) -> None:
    """Contexts long enough for splits, of which a lane's short one leaves most empty; the last split's nodes across
    its tiles' edge."""
    for heads, kvh, hd, t, base in ((16, 4, 128, 1, [9000, 5]), (32, 2, 256, 2, [4090]), (8, 2, 64, 30, [6000, 2001]),
                                    (32, 2, 256, 9, [5003, 77])):
        tree = tree_inputs.batch(["gaps" if t > 4 else "random"] * len(base), t)
        check(dev, *case(t, len(base), t, heads, kvh, hd, base), hd**-0.5, tree)


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(8, 2, 64, 4, [40]), (16, 4, 128, 20, [100, 3]), (32, 2, 256, 6, [3000])])
def test_a_chain_is_the_causal_order(dev, heads, kvh, hd, t, base) -> None:
    """Both calls are within their bars of the same 64-bit values, so within two of them of each other: their sums run in
    different orders."""
    q, k, v, table, b0 = case(t, len(base), t, heads, kvh, hd, base)
    got = check(dev, q, k, v, table, b0, hd**-0.5, tree_inputs.batch(["chain"] * len(base), t))
    want, spread = masked_attention_ref.paged_attention_masked(q, k, v, table, b0, hd**-0.5)
    assert float(((got - want).abs() / bars(want, spread)).max()) <= 1.0
    args = (q.to(dev), k.to(dev), attention.v_blocks(v).to(dev), table.to(dev), b0.to(dev), max(base) + t, hd**-0.5)
    other = attention.paged_attention_masked(*args).double().cpu()
    assert float(((got - other).abs() / bars(want, spread)).max()) <= 2.0


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(8, 2, 64, 4, [40]), (16, 4, 128, 20, [100, 3]), (32, 2, 256, 16, [3000, 64]),
                                                 (32, 2, 256, 2, [31])])
@pytest.mark.parametrize("worst", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min])
def test_what_a_node_does_not_see(dev, heads, kvh, hd, t, base, worst) -> None:
    """A node's key and value spoil the rows below it alone, and those behind the tree, in other blocks of the pool and of
    absent nodes nobody's; a spoilt query stays with its row."""
    q, k, v, table, b0 = case(t, len(base), t, heads, kvh, hd, base)
    tree = tree_inputs.batch(["random"] * len(base), t)
    tree[:, -1] = -2
    clean = run(dev, q, k, v, table, b0, hd**-0.5, tree)
    used = torch.zeros(k.shape[0], dtype=torch.bool)
    spoilt = t // 2  # a node of lane 0
    for j in range(len(base)):
        pos = torch.arange(base[j] + t - 1)
        used[table[j].long()[pos // 16] * 16 + pos % 16] = True
    at = base[0] + spoilt
    row = int(table[0, at // 16]) * 16 + at % 16
    for x in (k, v):
        x[~used] = worst
        x[row] = worst
    q[0, -1] = worst
    got = run(dev, q, k, v, table, b0, hd**-0.5, tree)
    below = torch.tensor([w is not None and spoilt in w for w in tree_ref.ways(tree[0])])
    keep = torch.ones(len(base), t, dtype=torch.bool)
    keep[0] = ~below
    off = (got.double() - clean.double()).abs().cpu()[keep]
    # the rows of a tile that holds such a value are done again in another order: their roundings alone differ
    assert float((off - 2.0**-7 * clean.double().abs().cpu()[keep]).max()) <= 2e-2
    assert not got[0, -1].any() and not bool(got.cpu()[keep].isnan().any())
    if worst != worst:
        assert bool(got[0].cpu()[below].isnan().all())


def test_strides_types_and_shared_trees(dev) -> None:
    heads, kvh, hd, t, base = 8, 2, 64, 9, [70, 3]
    q, k, v, table, b0 = case(4, 2, t, heads, kvh, hd, base)
    gate = torch.randn(2, t, heads, hd, generator=torch.Generator().manual_seed(1)).bfloat16()
    one = tree_inputs.batch(["random"], t)
    want = check(dev, q, k, v, table, b0, 0.2, one.expand(2, t), gate=gate)
    qg = torch.stack([q, gate], 3).flatten(3).to(dev)  # query and gate of a head side by side
    wide = torch.full((2, 3 * t), 99, dtype=torch.int64, device=dev)
    wide[:, ::3] = one.to(dev)
    args = (k.to(dev), attention.v_blocks(v).to(dev), table.long().to(dev), b0.int().to(dev), 96)
    for tree in (one.to(dev).expand(2, t), wide[:, ::3], one.to(dev).t().contiguous().t().expand(2, t)):
        got = attention.paged_attention_tree(qg[..., :hd], *args, 0.2, tree, gate=qg[..., hd:])
        assert torch.equal(got.double().cpu(), want)
    odd = torch.empty(2, t, heads, hd + 1, dtype=torch.bfloat16, device=dev)[..., 1:]  # rows off 16 bytes
    odd.copy_(qg[..., :hd])
    assert torch.equal(attention.paged_attention_tree(odd, *args, 0.2, one.to(dev).expand(2, t), gate=qg[..., hd:]).double().cpu(), want)


def test_past_the_table_and_bad_blocks(dev) -> None:
    """Positions past the table are not seen; a block outside the pool reads as zeros."""
    q, k, v, table, b0 = case(3, 2, 8, 8, 2, 64, [30, 30], spare=0)
    tree = tree_inputs.batch(["chain", "chain"], 8)
    short = table[:, :2]
    check(dev, q, k, v, short, b0, 0.1, tree, ctx=32)
    bad = table.clone()
    bad[0, 0], bad[1, 2] = -5, 2**31 - 1
    k0, v0 = k.clone(), v.clone()
    zero = torch.zeros(16, 2, 64, dtype=torch.bfloat16)
    got = run(dev, q, k, v, bad, b0, 0.1, tree).double().cpu()
    want, spread = tree_ref.attention(q, torch.cat([k0, zero]), torch.cat([v0, zero]), torch.where((bad < 0) | (bad > 99), k.shape[0] // 16, bad),
                                      b0, 0.1, tree)
    assert float(((got - want).abs() / bars(want, spread)).max()) <= 1.0


@pytest.mark.parametrize("seed", range(12))
def test_any_mix(dev, seed) -> None:
    r = random.Random(seed)
    heads, kvh, hd = r.choice(LAYOUTS)
    t, b = r.randint(1, 64), r.randint(1, 3)
    base = [r.randint(0, r.choice((20, 300, 1500))) for _ in range(b)]
    tree = tree_inputs.batch([r.choice(tree_inputs.SHAPES) for _ in range(b)], t, seed)
    gate = torch.randn(b, t, heads, hd, generator=torch.Generator().manual_seed(seed)).bfloat16() if r.random() < 0.5 else None
    check(dev, *case(seed, b, t, heads, kvh, hd, base), hd**-0.5, tree, gate=gate)


def test_in_a_graph_and_on_another_stream(dev) -> None:
    q, k, v, table, b0 = (x.to(dev) for x in case(8, 2, 12, 32, 2, 256, [900, 40]))
    vt, tree = attention.v_blocks(v), tree_inputs.batch(["random", "gaps"], 12).to(dev)
    call = lambda: attention.paged_attention_tree(q, k, vt, table, b0, 912, 0.06, tree)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        q.mul_(-0.9)
        tree.copy_(tree_inputs.batch(["random", "deep"], 12, i))
        b0.sub_(7)
        graph.replay()
        assert torch.equal(got, call())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, call())
