"""Trees of drafts on the CPU: their masks, depths and acceptance against the oracle, the model's rounds against greedy decode,
and the refusals that need no device."""

from __future__ import annotations

import ctypes

import pytest
import torch

import _mtpk
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


# ---------------------------------------------------------------- the C entry points: refused before anything is launched

P = 1 << 20  # an address that no refused call follows


@pytest.fixture(scope="module")
def lib():
    if not _mtpk.LIB_PATH.exists():
        import __graft_entry__

        __graft_entry__.build()
    return _mtpk.lib()


def array(kind, values) -> tuple:
    held = (kind * len(values))(*values)
    return ctypes.addressof(held), held


def refuse(entry, good: dict, bad: list[dict]) -> None:
    for change in bad:
        assert change.keys() <= good.keys()
        assert entry(*{**good, **change}.values(), None) == _mtpk.EINVAL, change


PAIR, PAIR_HELD = array(ctypes.c_int64, (4, 1))
QS, QS_HELD = array(ctypes.c_int64, (1024, 64, 256))


def test_attention_entry_refuses(lib) -> None:
    good = {"q": P, "qs": QS, "gate": None, "gs": QS, "b": 2, "t": 4, "heads": 4, "kvh": 2, "hd": 64, "k": P, "v": P, "rows": 160, "table": P,
            "stride": 5, "base": P, "scale": 0.1, "parents": P, "pdt": _mtpk.I32, "ps": PAIR, "n": 1, "ws": None, "wsb": 0, "out": P, "os": QS}
    refuse(lib.mtpk_paged_attention_tree, good, [
        *({n: None} for n in ("q", "qs", "k", "v", "table", "base", "parents", "ps", "out", "os")), {"gate": P, "gs": None}, {"t": 0}, {"t": 65},
        {"pdt": _mtpk.BF16}, {"b": -1}, {"heads": 3}, {"heads": 0}, {"kvh": 0}, {"hd": 96}, {"rows": 150}, {"rows": 0}, {"stride": 0}, {"scale": 0.0},
        {"scale": float("nan")}, {"n": 0}, {"n": 65}, {"n": 2}, {"heads": 65536, "kvh": 1}, {"q": P + 2},
        *({"b": (1 << 19) - 1, "t": 64, "heads": 1, "kvh": 1, "n": n, "ws": P, "wsb": 1 << 50} for n in (2, 8, 9, 64)),  # the merge's grid
    ])  # fmt: skip
    assert lib.mtpk_attention_tree_splits(2, 65, 8, 2, 64, 100) == 0
    assert lib.mtpk_attention_tree_splits(2, 4, 8, 2, 64, 0) == 1
    assert lib.mtpk_attention_tree_workspace_bytes(2, 65, 8, 2, 64, 4) == 0


def test_delta_net_entries_refuse(lib) -> None:
    good = {"proj": P, "dt": _mtpk.BF16, "stride": 200, "conv": P, "slot": P, "slots": 3, "w": P, "a_log": P, "bias": P, "parents": P,
            "pdt": _mtpk.I64, "ps": PAIR, "b": 2, "t": 4, "kh": 1, "kd": 16, "vh": 2, "vd": 16, "taps": 4, "eps": 1e-6, "scale": 0.25, "q": P,
            "k": P, "v": P, "g": P, "beta": P}
    refuse(lib.mtpk_deltanet_prep_tree, good, [
        *({n: None} for n in ("proj", "conv", "slot", "w", "a_log", "bias", "parents", "ps", "q", "k", "v", "g", "beta")), {"dt": _mtpk.I32},
        {"pdt": _mtpk.F32}, {"t": 0}, {"t": 65}, {"b": -1}, {"b": 1 << 31}, {"kd": 257}, {"kd": 0}, {"vd": 300}, {"kh": 0}, {"vh": 65536}, {"taps": 1},
        {"taps": 10}, {"slots": 0}, {"stride": 99}, {"stride": 1 << 23},
    ])  # fmt: skip
    good = {"state": P, "slots": 3, "slot": P, "rows": 2, "t": 4, "heads": 4, "qk": 2, "kd": 16, "vd": 8, "q": P, "k": P, "v": P, "g": P, "beta": P,
            "parents": P, "pdt": _mtpk.I32, "ps": PAIR, "out": P}
    shapes = [{"t": 0}, {"t": 65}, {"rows": -1}, {"heads": 3}, {"heads": 0}, {"qk": 0}, {"kd": 48}, {"vd": 0}, {"vd": 4097}, {"slots": 0},
              {"slots": 1 << 40}, {"rows": 1 << 40}]
    refuse(lib.mtpk_delta_rule_tree, good, [
        *shapes, *({n: None} for n in ("state", "q", "k", "v", "g", "beta", "parents", "ps", "out")), {"pdt": 9}, {"slot": None, "rows": 4},
    ])  # fmt: skip
    good = {"state": P, "slots": 3, "slot": P, "rows": 2, "t": 4, "heads": 4, "qk": 2, "kd": 16, "vd": 8, "k": P, "v": P, "g": P, "beta": P,
            "path": P, "lengths": P, "conv": P, "cdt": _mtpk.F32, "cslots": 3, "proj": P, "stride": 64, "channels": 64, "k1": 3}
    refuse(lib.mtpk_deltanet_commit_path, good, [
        *shapes, *({n: None} for n in ("state", "slot", "k", "v", "g", "beta", "path", "lengths", "conv", "proj")), {"cdt": _mtpk.I64}, {"cslots": 0},
        {"stride": 63}, {"channels": 0}, {"k1": 0}, {"k1": 9},
    ])  # fmt: skip


def test_acceptance_and_move_entries_refuse(lib) -> None:
    outs = ("path", "n", "lengths", "keep", "bonus", "next", "left", "live", "src")
    good = {"best": P, "bs": 4, "tokens": P, "ts": 4, "parents": P, "pdt": _mtpk.I32, "ps": PAIR, "active": P, "pos": P, "budget": P, "stops": P,
            "n_stops": 2, "b": 2, "t": 4, **dict.fromkeys(outs, P)}
    refuse(lib.mtpk_tree_accept, good, [
        *({n: None} for n in ("best", "tokens", "parents", "ps", "active", "pos", "budget", "stops", *outs)), {"t": 0}, {"t": 65}, {"b": -1},
        {"b": 1 << 40}, {"n_stops": -1}, {"pdt": _mtpk.F32},
    ])  # fmt: skip

    def pools(ps=(P, P + (1 << 20)), channels=(16, 16), size=(2, 2), transposed=(0, 1)) -> tuple[dict, list]:
        made = {"pools": array(ctypes.c_void_p, ps), "channels": array(ctypes.c_int64, channels), "size": array(ctypes.c_int, size),
                "transposed": array(ctypes.c_int, transposed)}
        return {n: x[0] for n, x in made.items()}, [x[1] for x in made.values()]

    first, held = pools()
    good = {**first, "n": 2, "blocks": 8, "table": P, "stride": 2, "base": P, "path": P, "lengths": P, "b": 2, "t": 4}
    refuse(lib.mtpk_keep_path, good, [
        *({n: None} for n in ("pools", "channels", "size", "transposed", "table", "base", "path", "lengths")), {"n": 0}, {"blocks": 0}, {"stride": 0},
        {"stride": 1 << 27}, {"t": 0}, {"t": 65}, {"b": -1},
    ])  # fmt: skip
    for change in ({"ps": (P, P)}, {"ps": (P, P + 4080)}, {"ps": (P + 4080, P)}, {"ps": (P, P + (1 << 20) + 8)}, {"ps": (P, 0)}, {"channels": (4, 16)},
                   {"channels": (16, 0)}, {"size": (2, 8)}):
        made, held2 = pools(**change)
        refuse(lib.mtpk_keep_path, good, [made])
    assert held and held2
