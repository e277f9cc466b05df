"""DeltaNet rows of trees of drafts (`prep_tree`, `delta_rule_tree`, `commit_path`) against the 64-bit oracle.

Bars of the rule as in test_gpu_deltanet_steps: sums of fp32 products with decays of at most 1 and keys of at most unit
length, 1e-5 of the largest value, about 100 fp32 roundings. Of the preparation: fp32's exponentials, roots and sums of 256
squares are off by a few 2^-24 of a value (2e-6 allowed); a bf16 convolution is the rounded exact value itself."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import deltanet
from oracle import tree_ref
from tests import tree_inputs

from .test_gpu_deltanet import _case, _dev

pytestmark = pytest.mark.gpu


def _close(got, want):
    assert np.abs(got - want).max() <= 1e-5 * max(np.abs(want).max(), 1e-30), np.abs(got - want).max() / np.abs(want).max()


SHAPES = [  # heads, q/k heads, k_dim, v_dim
    (4, 2, 16, 16), (3, 3, 32, 96), (2, 1, 64, 64), (4, 1, 128, 128), (3, 1, 128, 64), (5, 5, 128, 192), (2, 2, 128, 40), (8, 2, 64, 128),
    (2, 1, 16, 18), (2, 1, 128, 70), (1, 1, 64, 33), (3, 1, 32, 1),  # columns in no groups of four
]


@pytest.mark.parametrize("heads,qk,dk,dv", SHAPES)
@pytest.mark.parametrize("t,kinds", [(1, ["chain"]), (2, ["star", "empty"]), (7, ["random", "gaps", "forest"]), (16, ["deep", "random"]),
                                     (17, ["gaps"]), (33, ["random", "chain"]), (48, ["gaps", "random"]), (49, ["forest"]), (61, ["random"]), (64, ["deep", "gaps"])])
def test_rule(dev, heads, qk, dk, dv, t, kinds) -> None:
    b = len(kinds)
    pool, slots, q, k, v, g, beta = _case(t + dk + heads, b + 2, heads, qk, dk, dv, b, t)
    g[:, ::3] *= 20  # decays that forget the state, next to ones that keep it
    tree = tree_inputs.batch(kinds, t)
    args = _dev(dev, pool, slots.astype(np.int64), q, k, v, g, beta)
    got = deltanet.delta_rule_tree(*args, tree.to(dev)).cpu().numpy()
    _close(got, tree_ref.delta_rule(pool, slots, q, k, v, g, beta, tree))
    absent = np.array([[w is None for w in tree_ref.ways(p)] for p in tree])
    assert not got[absent].any()
    assert torch.equal(args[0].cpu(), torch.from_numpy(pool))  # the states are read alone


def test_rule_slots(dev) -> None:
    pool, _, q, k, v, g, beta = _case(5, 4, 4, 2, 128, 128, 3, 9)
    tree = tree_inputs.batch(["random"] * 3, 9, dtype=torch.int64)
    args = _dev(dev, pool, q, k, v, g, beta)
    want = tree_ref.delta_rule(pool, range(3), q, k, v, g, beta, tree)
    _close(deltanet.delta_rule_tree(args[0], None, *args[1:], tree.to(dev)).cpu().numpy(), want)
    got = deltanet.delta_rule_tree(args[0], torch.tensor([0, 9, -1], device=dev), *args[1:], tree.to(dev)).cpu().numpy()
    _close(got[0], want[0])
    assert not got[1:].any()


def test_rule_on_a_chain(dev) -> None:
    pool, slots, q, k, v, g, beta = _case(3, 5, 8, 2, 128, 128, 3, 12)
    args = _dev(dev, pool, slots.astype(np.int64), q, k, v, g, beta)
    got = deltanet.delta_rule_tree(*args, tree_inputs.batch(["chain"] * 3, 12).to(dev))
    _close(got.cpu().numpy(), deltanet.delta_rule(*args).cpu().numpy().astype(np.float64))


@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (32, 40)])
@pytest.mark.parametrize("what", ["nan_k", "nan_v", "inf_v", "inf_q", "long_k", "growing", "minus_inf_g", "beta", "nan_state", "large_state",
                                  "overflow"])
def test_rule_with_values_out_of_range(dev, what, dk, dv) -> None:
    """What is not finite reaches a node's own descendants (or all nodes, from the state), no other; what is finite and
    outside the layer's range is computed all the same."""
    t, bad = 20, 6
    pool, slots, q, k, v, g, beta = _case(8, 3, 4, 4, dk, dv, 2, t)
    tree = tree_inputs.batch(["random", "random"], t)
    args = [torch.from_numpy(np.ascontiguousarray(x)) for x in (pool, slots.astype(np.int64), q, k, v, g, beta)]
    plain = deltanet.delta_rule_tree(*(x.to(dev) for x in args), tree.to(dev)).cpu()
    ps, _, pq, pk, pv, pg, pb = args
    if what == "nan_k":
        pk[1, bad, 2, 5] = np.nan
    elif what == "nan_v":
        pv[1, bad, 2, 7] = np.nan
    elif what == "inf_v":
        pv[1, bad, 2, 7] = np.inf
    elif what == "inf_q":
        pq[1, bad, 2, 3] = np.inf
    elif what == "long_k":
        pk[1, bad, 2] *= 3
    elif what == "growing":
        pg[1, bad, 2] = 2.5
    elif what == "minus_inf_g":
        pg[1, bad, 2] = -np.inf
    elif what == "beta":
        pb[1, bad, 2] = 1.9
    elif what == "nan_state":
        ps[slots[1], 2, 3, 7] = np.nan
    elif what == "large_state":
        ps[slots[1], 2, 3, 7] = 1e32
    elif what == "overflow":
        pv[1, bad, 2, 7] = 3e38
        pv[1, bad + 1 :, 2, 7] = -3e38
    got = deltanet.delta_rule_tree(*(x.to(dev) for x in args), tree.to(dev)).cpu()
    below = torch.tensor([bad in w for w in tree_ref.ways(tree[1])])
    hit = torch.zeros(2, t, 4, dv, dtype=torch.bool)
    if what in ("nan_v", "inf_v"):
        hit[1, below, 2, 7] = True
    elif what == "inf_q":
        hit[1, bad, 2] = True
    elif what in ("nan_state", "large_state"):
        hit[1, :, 2, 7] = True
    elif what == "overflow":
        hit[1, bad:, 2, 7] = True
    else:
        hit[1, below, 2] = True
    assert bool(got[~hit].isfinite().all())
    _close(got[~hit].numpy(), plain[~hit].numpy().astype(np.float64))
    if what in ("nan_k", "nan_v", "nan_state", "inf_q", "inf_v"):
        assert not bool(got[hit].isfinite().any())
    elif what == "overflow":
        pass
    else:
        want = torch.from_numpy(tree_ref.delta_rule(*(x.numpy() for x in args), tree))
        off = (got.double() - want).abs()
        column = want.abs().amax((1, 3), keepdim=True)  # a (row, head)'s own scale
        assert float((off / column).max()) <= 1e-5


def _silu64(x):
    return x / (1 + np.exp(-x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kh,kd,vh,vd,taps", [(2, 128, 4, 128, 4), (1, 16, 2, 16, 4), (3, 40, 2, 250, 4), (2, 33, 3, 17, 4), (1, 64, 1, 64, 2),
                                              (2, 24, 2, 8, 9), (1, 200, 2, 128, 3)])
@pytest.mark.parametrize("t,kinds", [(1, ["chain", "chain"]), (6, ["random", "gaps"]), (23, ["forest", "deep", "empty"]), (64, ["random"])])
def test_prep(dev, dtype, kh, kd, vh, vd, taps, t, kinds) -> None:
    g = torch.Generator().manual_seed(t + kd + taps)
    b, C = len(kinds), 2 * kh * kd + vh * vd
    proj = torch.randn(b, t, C + vh * vd + 2 * vh + 3, generator=g).to(dtype)
    conv = torch.randn(b + 2, C, taps - 1, generator=g).to(dtype)
    w = (torch.randn(C, taps, generator=g) * 0.4).to(dtype)
    a_log, dt_bias = torch.randn(vh, generator=g), torch.randn(vh, generator=g)
    slots = torch.randperm(b + 2, generator=g)[:b]
    if b > 1:
        slots[1] = 77  # no slot: a zero window
    tree = tree_inputs.batch(kinds, t)
    got = deltanet.prep_tree(*(x.to(dev) for x in (proj, conv, slots, w, a_log, dt_bias)), kh, kd, vh, vd, tree.to(dev))
    acc = tree_ref.conv_rows(conv.double().numpy(), slots, w.double().numpy(), proj[..., :C].double().numpy(), tree)
    y = torch.from_numpy(_silu64(acc)).to(dtype).double()
    q, k = (y[..., i * kh * kd : (i + 1) * kh * kd].view(b, t, kh, kd) for i in range(2))
    v = y[..., 2 * kh * kd :].view(b, t, vh, vd)
    q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    z = C + vh * vd
    beta = torch.sigmoid(proj[..., z : z + vh].double())
    decay = -a_log.double().exp() * torch.nn.functional.softplus(proj[..., z + vh : z + 2 * vh].double() + dt_bias.double(), threshold=1e9)
    present = torch.tensor([[x is not None for x in tree_ref.ways(p)] for p in tree])
    for x, want in zip(got, (q * kd**-0.5, k, v, decay, beta), strict=True):
        x = x.double().cpu()
        assert not x[~present].any()
        want = want * present.view(b, t, *[1] * (want.dim() - 2))
        # f32: sums of up to nine products that may cancel, 9 * 2^-24 of the largest terms each
        room = 4e-6 * want.abs() + (1e-5 if dtype == torch.float32 else 1e-7) * max(float(want.abs().max()), 1e-30)
        assert bool(((x - want).abs() <= room).all())


def test_prep_on_a_chain_and_strided_rows(dev) -> None:
    """f32 rows of a chain are `prep`'s: v, g and beta bit for bit. q and k are up to the order in which 128 squares are
    summed, which `prep` itself chooses by size: a sum of positive terms is off by at most its 8 roundings (a square, a sum
    in the lane, six between lanes), two sums by 16, of which the root leaves 8, and three roundings follow on either
    side: 14 * 2^-24. Rows with room between them are read in place."""
    g = torch.Generator().manual_seed(2)
    kh, kd, vh, vd, b, t = 2, 128, 4, 128, 3, 7
    C = 2 * kh * kd + vh * vd
    P = C + vh * vd + 2 * vh
    proj, conv, w = (torch.randn(*s, generator=g).to(dev) for s in ((b, t, P), (b, C, 3), (C, 4)))
    rest = (torch.randn(vh, generator=g).to(dev), torch.randn(vh, generator=g).to(dev), kh, kd, vh, vd)
    slots, tree = torch.arange(b, device=dev), tree_inputs.batch(["chain"] * b, t).to(dev)
    got = deltanet.prep_tree(proj, conv, slots, w, *rest, tree)
    want = deltanet.prep(proj, conv, slots, w, *rest)
    assert all(torch.equal(x, y) for x, y in zip(got[2:], want[2:]))
    assert all(bool(((x - y).abs() <= 14 * 2.0**-24 * y.abs()).all()) for x, y in zip(got[:2], want[:2]))
    for dtype in (torch.float32, torch.bfloat16):
        args = conv.to(dtype), slots, w.to(dtype)
        want = deltanet.prep_tree(proj.to(dtype), *args, *rest, tree)
        wide = torch.empty(b, t, P + 5, dtype=dtype, device=dev)
        wide[..., :P] = proj
        apart = torch.empty(b, 2 * t, P, dtype=dtype, device=dev)  # lanes' rows at no one stride
        apart[:, :t] = proj
        for x in (wide[..., :P], apart[:, :t]):
            assert all(torch.equal(u, v) for u, v in zip(deltanet.prep_tree(x, *args, *rest, tree), want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,qk,dk,dv,t", [(4, 2, 16, 16, 5), (3, 1, 32, 96, 4), (4, 2, 128, 128, 9), (2, 2, 128, 64, 64), (2, 1, 128, 40, 6),
                                              (2, 1, 64, 64, 1)])
@pytest.mark.parametrize("k1", [3, 1, 8])
def test_commit(dev, heads, qk, dk, dv, t, k1, dtype) -> None:
    b = 5
    pool, slots, q, k, v, g, beta = _case(t + dk, b + 3, heads, qk, dk, dv, b, t)
    r = np.random.default_rng(t)
    lengths = np.array([t, max(t // 2, 1), 1, 0, t + 3])
    path = np.stack([np.sort(np.concatenate([[0], r.permutation(np.arange(1, t))])) for _ in range(b)])
    for j in range(1, b):  # some nodes, rising, the last one repeated
        n = min(max(int(lengths[j]), 1), t)
        some = np.sort(np.concatenate([[0], r.permutation(np.arange(1, t))[: n - 1]]))
        path[j] = np.concatenate([some, np.full(t - n, some[-1])])
    if t > 4:
        path[4, 2:] = [-1, t, 2**40][t % 3]  # ends the path
    slots[2] = [-1, b + 3][t % 2]
    C = 70
    raw, conv = torch.from_numpy(r.standard_normal((b, t, C + 9))).to(dtype), torch.from_numpy(r.standard_normal((b + 3, C, k1))).to(dtype)
    state, ts, tk, tv, tg, tb, tp, tl = _dev(dev, pool, slots.astype(np.int64), k, v, g, beta, path, lengths)
    win = conv.to(dev)
    deltanet.commit_path(state, win, ts, tk, tv, tg, tb, tp, tl, raw.to(dev), C)
    want, columns = tree_ref.commit(pool, conv.double().numpy(), slots, k, v, g, beta, path, lengths, raw[..., :C].double().numpy())
    _close(state.cpu().numpy(), want)
    assert np.array_equal(win.double().cpu().numpy(), columns)
    for s in set(range(b + 3)) - set(slots[[0, 1, 4]].tolist()):
        assert torch.equal(state[s].cpu(), torch.from_numpy(pool[s]))


def test_commit_of_a_prefix_is_the_chains(dev) -> None:
    pool, slots, q, k, v, g, beta = _case(3, 6, 8, 2, 128, 128, 4, 6)
    args = _dev(dev, pool, slots.astype(np.int64), q, k, v, g, beta)
    lengths = torch.tensor([1, 6, 3, 0], device=dev)
    proj, conv = torch.randn(4, 6, 300, device=dev), torch.randn(6, 256, 3, device=dev)
    one, win = args[0].clone(), conv.clone()
    idx = (lengths[:, None] + torch.arange(3, device=dev)).clamp(max=8)
    deltanet.commit(one, win, *args[1:], lengths, proj, idx, 256)
    deltanet.commit_path(args[0], conv, args[1], *args[3:], torch.arange(6, device=dev).expand(4, 6), lengths, proj, 256)
    assert torch.equal(one, args[0]) and torch.equal(win, conv)


def test_in_a_graph(dev) -> None:
    pool, slots, q, k, v, g, beta = _case(3, 6, 8, 2, 128, 128, 3, 10)
    args = _dev(dev, pool, slots.astype(np.int64), q, k, v, g, beta)
    tree = tree_inputs.batch(["random", "gaps", "deep"], 10).to(dev)
    C = 256 * 2 + 8 * 128
    proj, conv, w = (torch.randn(*s, device=dev).bfloat16() for s in ((3, 10, C + 8 * 128 + 16), (6, C, 3), (C, 4)))
    rest = (torch.zeros(8, device=dev), torch.zeros(8, device=dev), 2, 128, 8, 128)
    path = torch.arange(10, device=dev).repeat(3, 1)
    lengths = torch.tensor([1, 4, 2], device=dev)

    def step(state, window):
        made = deltanet.prep_tree(proj, window, args[1], w, *rest, tree)
        out = deltanet.delta_rule_tree(state, args[1], *made, tree)
        deltanet.commit_path(state, window, args[1], *made[1:], path, lengths, proj, C)
        return out

    mine, eager = (args[0].clone(), conv.clone()), (args[0].clone(), conv.clone())
    step(args[0].clone(), conv.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*mine)
    for i in range(4):
        proj.mul_(-0.9)
        tree.copy_(tree_inputs.batch(["random", "star", "gaps"], 10, i))
        lengths.add_(1)
        graph.replay()
        assert torch.equal(got, step(*eager))
        assert all(torch.equal(x, y) for x, y in zip(mine, eager))
