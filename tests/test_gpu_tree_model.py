"""The operators of a tree together, as the model's verify round runs them: forward, acceptance, and the commit of cache rows,
states and windows, on the device."""

from __future__ import annotations

import pytest
import torch

import attention
import graph_mtp
import mtp
import verify_model as vm
from oracle import tree_ref
from tests import model_helpers as mh
from tests import tree_inputs, tree_round

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,t", [("chain", 4), ("star", 7), ("random", 16), ("deep", 9), ("random", 1)])
def test_rounds_match_greedy(dev, kind, t) -> None:
    """The fp32 model on the device: rounds over trees commit what plain decode on the CPU commits."""
    ids, steps = mh.prompts(), 24
    truth = mh.greedy_truth(mh.build(), ids, steps + 20)
    model = mh.build(dev)
    for lane, p in enumerate(ids):
        model.prefill(lane, p)
    at, rnd = [0, 0], 0
    while min(at) < steps:
        lanes = [j for j in range(2) if at[j] < steps]
        trees = [tree_round.planted(kind, t, truth[j][at[j] : steps + 1], model.cfg.vocab, 10 * rnd + j) for j in lanes]
        tokens, parents = [x[0] for x in trees], [x[1] for x in trees]
        left = [steps - at[j] for j in lanes]
        out = tree_round.run(model, lanes, tokens, parents, [16 + at[j] for j in lanes], 96, budget=left)
        for i, j in enumerate(lanes):
            got = tree_round.committed(out, tokens, i)
            assert len(got) >= min(trees[i][2] + 1, left[i])
            assert got == truth[j][at[j] + 1 : at[j] + 1 + len(got)]
            at[j] += len(got)
        rnd += 1
    seq = mh.build(dev)
    for lane, p in enumerate(ids):
        seq.prefill(lane, p)
        vm.greedy_reference(seq, lane, truth[lane][0], 16, at[lane])
        mh.assert_slot_state_close(model, seq, lane, 16 + at[lane], rtol=1e-4, atol=1e-5)


def real_layers(dev, lanes: int, start: int) -> vm.Model:
    """Real layer dimensions in bf16, each lane with `start` positions of seeded context."""
    model = vm.Model(vm.verify_cfg(), dev, torch.bfloat16, lanes=lanes, max_seq=start + 128, seed=0, expert_mode="bytes",
                     moe_rows=lanes * 16)
    mtp.attach(model, k=3, seed=1, expert_mode="bytes")
    g = torch.Generator(device=dev).manual_seed(3)
    for lane in range(lanes):
        model.blocks.grow(lane, start)
    for ty, pool in zip(model.cfg.layer_types, model.pool, strict=True):
        if ty == vm.ATTN:
            pool["k"].normal_(generator=g), pool["v"].normal_(generator=g)
        else:
            pool["conv"].normal_(generator=g), pool["rec"].normal_(0, 0.05, generator=g)
    model.mtp.pool["k"].normal_(generator=g), model.mtp.pool["v"].normal_(generator=g)
    model.hidden_cache.normal_(generator=g)
    return model


def model_path(model, lanes, tokens, pos, t, ctx) -> list[list[int]]:
    """Each lane's greedy continuation of t - 1 ids after `tokens`, as forwards of a growing chain choose them."""
    rows = [[x] for x in tokens]
    model.blocks.grow_many(lanes, [p + t for p in pos])
    for n in range(1, t):
        ids = torch.tensor(rows, device=model.device)
        res = model.forward_rows(ids, lanes, torch.tensor(pos, device=model.device), ctx, final_norm=True,
                                 parents=tree_inputs.batch(["chain"] * len(lanes), n).to(model.device))
        best = model.next_tokens(res.normed[:, -1].contiguous()).view(-1).tolist()
        for row, x in zip(rows, best, strict=True):
            row.append(x)
    return rows


def test_a_round_at_real_sizes_captured_and_replayed(dev) -> None:
    """bf16 layers of the real sizes: the round captured in a graph and replayed leaves, replay after replay, what the eager
    round leaves, bit for bit, and the lane that is not active as it was."""
    lanes, t, start = [0, 1, 2], 12, 300
    model = real_layers(dev, 3, start + t)
    toks, pos = [5, 900, 77], [start, start - 7, start + 5]
    ctx = start + 5 + t
    truth = model_path(model, lanes, toks, pos, 5, ctx)
    trees = [tree_round.planted("random", t, truth[j], model.cfg.vocab, j) for j in range(3)]
    on = lambda x, dtype=torch.int64: torch.tensor(x, dtype=dtype, device=dev)  # noqa: E731
    model.blocks.grow_many(lanes, [p + t for p in pos])
    args = (on(lanes), on([x[0] for x in trees]), on([x[1] for x in trees], torch.int32), on(pos), on([9, 9, 9]),
            torch.full((3, 2), -1, device=dev))
    active = on([1, 0, 1], torch.bool)
    table = model.blocks.table[args[0]]

    def step() -> graph_mtp.TreeAccept:
        return graph_mtp.verify_tree(model, *args, ctx, active=active, block_table=table)

    before = mh.snapshot(model)
    out = step()
    names = ("path", "accept_len", "lengths", "keep", "bonus", "next_pos", "budget_left", "live", "hidden_src")
    want, after = [getattr(out, n).clone() for n in names], mh.snapshot(model)
    lane1 = mh.slot_state(model, 1, pos[1])
    mh.restore(model, before)
    assert all(torch.equal(x, y) for x, y in zip(mh.slot_state(model, 1, pos[1]), lane1, strict=True))
    step()
    mh.restore(model, before)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        mh.restore(model, before)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(getattr(got, n), x) for n, x in zip(names, want, strict=True))
        ends = [pos[lane] + int(n) for lane, n in enumerate(want[2].tolist())]
        left = [mh.slot_state(model, lane, ends[lane]) for lane in (0, 2)]
        mh.restore(model, after)
        for lane, mine in zip((0, 2), left, strict=True):
            assert all(torch.equal(x, y) for x, y in zip(mine, mh.slot_state(model, lane, ends[lane]), strict=True))
        mh.restore(model, before)
        step()  # eager work between replays


def test_a_commit_at_real_sizes_is_the_chain_s_of_the_path(dev) -> None:
    """bf16 layers of the real sizes: what `commit_path` leaves is bit for bit what `commit` leaves of the path's rows in order,
    and the cache rows are the ones that the forward wrote for the path."""
    t, start = 16, 200
    model = real_layers(dev, 2, start + t)
    g = torch.Generator().manual_seed(1)
    pos, lanes = torch.tensor([start, start - 9], device=dev), torch.tensor([0, 1], device=dev)
    model.blocks.grow_many([0, 1], [start + t, start - 9 + t])
    tree = tree_inputs.batch(["random", "deep"], t, 4).to(dev)
    tokens = torch.randint(0, model.cfg.vocab, (2, t), generator=g).to(dev)
    res = model.forward_rows(tokens, lanes, pos, start + t, parents=tree)
    ways = [max((w for w in tree_ref.ways(p) if w), key=len) for p in tree.tolist()]
    lengths = torch.tensor([len(w) for w in ways], device=dev)
    path = torch.tensor([w + w[-1:] * (t - len(w)) for w in ways], device=dev)
    at = torch.arange(2, device=dev)[:, None]
    written = model.blocks.physical_rows(lanes, pos[:, None] + path)
    rows = [(p["k"][written], attention.read_v(p["v"], written.reshape(-1))) for p in model.pool if "k" in p]
    before = mh.snapshot(model)
    for i, r in res.dn_rows.items():
        chain = vm.DeltaNetRows(r.proj[at, path][..., : model.cfg.conv_dim].transpose(1, 2),
                                *(x[at, path].contiguous() for x in (r.q, r.k, r.v, r.g, r.beta, r.proj)))
        model.deltanet_commit(model.pool[i], chain, lanes, lengths)
    want = {i: (model.pool[i]["rec"].clone(), model.pool[i]["conv"].clone()) for i in res.dn_rows}
    mh.restore(model, before)
    model.commit_path(res, lanes, pos, path, lengths)
    for i, (rec, conv) in want.items():
        assert torch.equal(model.pool[i]["rec"], rec) and torch.equal(model.pool[i]["conv"], conv)
    kept = model.blocks.physical_rows(lanes, pos[:, None] + torch.arange(t, device=dev))
    for p, (k, v) in zip((p for p in model.pool if "k" in p), rows, strict=True):
        now = attention.read_v(p["v"], kept.reshape(-1)).view(2, t, *v.shape[1:])
        for j in range(2):
            n = len(ways[j])
            assert torch.equal(p["k"][kept][j, :n], k[j, :n]) and torch.equal(now[j, :n], v.view_as(now)[j, :n])
