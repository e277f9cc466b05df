"""Forked, trimmed and compacted block tables, block copies on the CPU, and the C entry points' refusals."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

import _mtpk
import attention
import verify_model as vm
from tests import model_helpers


def _tables(lanes=5, max_seq=160, seed=0):
    return vm.BlockTables(lanes, max_seq, 16, torch.device("cpu"), seed=seed)


def _invariants(t):
    count = {}
    for lane, have in enumerate(t.host):
        assert len(set(have)) == len(have) and 0 not in have
        assert t.held_positions[lane] == 16 * len(have)
        assert t.table[lane].tolist() == have + [0] * (t.max_blocks - len(have))
        for block in have:
            count[block] = count.get(block, 0) + 1
    assert {b: n for b, n in count.items() if n > 1} == t._holders
    assert sorted(t._free) == sorted(set(range(1, t.n_blocks)) - set(count))


def test_fork_shares_whole_blocks_and_copies_the_last() -> None:
    t = _tables()
    t.grow(0, 70)
    src, dst = t.fork(0, 3, 40)
    assert t.host[3][:2] == t.host[0][:2] and (src, dst) == ([t.host[0][2]], [t.host[3][2]])
    assert t.host[3][2] not in t.host[0]
    assert t.fork(0, 4, 32) == ([], []) and t.host[4] == t.host[0][:2]
    _invariants(t)
    t.grow(4, 50)
    t.release(0)
    _invariants(t)
    t.release(4)
    t.release(3)
    _invariants(t)
    assert len(t._free) == t.n_blocks - 1
    t.grow(1, 16)
    assert t.fork(1, 2, 0) == ([], []) and t.host[2] == []
    for bad in (lambda: t.fork(1, 1, 3), lambda: t.fork(2, 1, 0), lambda: t.fork(1, 2, 17), lambda: t.fork(1, 2, -1)):
        with pytest.raises(ValueError):
            bad()
    _invariants(t)


def test_a_fork_without_a_free_block_changes_nothing() -> None:
    t = vm.BlockTables(2, 32, 16, torch.device("cpu"))
    t.grow(0, 32)
    t._free.clear()
    before = [list(h) for h in t.host]
    with pytest.raises(ValueError):
        t.fork(0, 1, 20)
    assert t.host == before and not t._holders


def test_trim() -> None:
    t = _tables()
    t.grow(0, 100)
    t.trim(0, 33)
    assert len(t.host[0]) == 3
    t.trim(0, 48)
    t.trim(0, 1000)
    assert len(t.host[0]) == 3
    _invariants(t)
    t.trim(0, 0)
    _invariants(t)
    with pytest.raises(ValueError):
        t.trim(0, -1)


def test_any_order_keeps_every_lanes_positions() -> None:
    """Grow, write, fork, trim, release and compact at random, with copies done as asked: every lane reads
    back what it wrote."""
    rng = random.Random(4)
    t = _tables(lanes=6, seed=2)
    k = torch.zeros(t.rows, 1, 2)
    v = torch.zeros(t.n_blocks, 1, 2, 16)
    kept = [[] for _ in range(6)]  # what each lane wrote, by position
    stamp = 0
    for _ in range(400):
        lane, other = rng.randrange(6), rng.randrange(6)
        act = rng.choice(("write", "write", "write", "fork", "trim", "release", "compact"))
        if act == "write" and len(kept[lane]) < 150:
            n = rng.randint(1, 9)
            if len(t._free) < 2:
                continue
            t.grow(lane, len(kept[lane]) + n)
            for _ in range(n):
                stamp += 1
                p = len(kept[lane])
                row = int(t.physical_rows(torch.tensor([lane]), torch.tensor([[p]]))[0, 0])
                k[row], v[row // 16, :, :, row % 16] = stamp, -stamp
                kept[lane].append(stamp)
        elif act == "fork" and lane != other and t._free:
            t.release(other)
            n = rng.randint(0, len(kept[lane]))
            attention.copy_blocks([k, v], *t.fork(lane, other, n))
            kept[other] = kept[lane][:n]
        elif act == "trim":
            n = rng.randint(0, len(kept[lane]))
            n -= n % 16  # a shared block's positions past n may be written by another lane from here on
            t.trim(lane, n)
            kept[lane] = kept[lane][:n]
        elif act == "release":
            t.release(lane)
            kept[lane] = []
        elif act == "compact":
            src, dst = t.compact()
            assert not set(src) & set(dst) and len(set(dst)) == len(dst)
            attention.copy_blocks([k, v], src, dst)
            held = {b for h in t.host for b in h}
            assert held == set(range(1, len(held) + 1))
        _invariants(t)
        for j, want in enumerate(kept):
            if want:
                rows = t.physical_rows(torch.tensor([j]), torch.arange(len(want))[None])[0]
                assert k[rows, 0, 0].tolist() == want and v[rows // 16, 0, 1, rows % 16].tolist() == [-x for x in want]


def test_trim_inside_a_shared_block_takes_one_of_its_own() -> None:
    """Lanes that share a block, one of them cut back into it: its next positions are its own."""
    for grown, keep in ((64, 40), (64, 63), (48, 40), (33, 7)):  # the last one with blocks between, and none let go
        t = _tables()
        t.grow(0, grown)
        assert t.fork(0, 1, grown // 16 * 16) == ([], [])
        before = list(t.host[0])
        src, dst = t.trim(1, keep)
        last = keep // 16
        assert src == [before[last]] and dst == [t.host[1][last]] and dst[0] not in before
        assert t.host[0] == before and t.host[1][:last] == before[:last]
        _invariants(t)
        t.grow(1, keep + 1)
        rows = t.physical_rows(torch.tensor([0, 1]), torch.tensor([[keep], [keep]]))
        assert int(rows[0, 0]) != int(rows[1, 0])
        assert t.trim(1, keep) == ([], [])  # its own by now
        assert t.trim(0, keep) == ([], [])  # the source holds it alone
        _invariants(t)
    t = _tables()
    t.grow(0, 32)
    t.fork(0, 1, 32)
    assert t.trim(1, 16) == ([], []) and t.host[1] == t.host[0][:1]  # whole blocks stay shared
    _invariants(t)


def test_trim_inside_a_shared_block_without_a_free_one() -> None:
    t = _tables(lanes=3, max_seq=64)
    t.grow(0, 48)
    t.fork(0, 1, 48)
    t._free.clear()
    before, table = [list(h) for h in t.host], t.table.clone()
    with pytest.raises(ValueError):
        t.trim(1, 20)
    assert t.host == before and torch.equal(t.table, table) and len(t._holders) == 3
    t = _tables(lanes=3, max_seq=64)
    t.grow(0, 48)
    t.fork(0, 1, 32)
    t.grow(1, 48)  # a third block of its own, which the cut gives back before it needs one
    t._free.clear()
    own = t.host[1][2]
    assert t.trim(1, 20) == ([t.host[0][1]], [own]) and t.host[1] == [t.host[0][0], own]


def test_any_order_with_cuts_inside_blocks_keeps_every_lanes_positions() -> None:
    """As above, with cuts at any position: what a lane writes after one is read by no other lane."""
    for seed in range(4):
        rng = random.Random(seed)
        t = _tables(lanes=6, seed=seed)
        k, v = torch.zeros(t.rows, 1, 2), torch.zeros(t.n_blocks, 1, 2, 16)
        kept = [[] for _ in range(6)]
        stamp = 0
        for _ in range(400):
            lane, other = rng.randrange(6), rng.randrange(6)
            act = rng.choice(("write", "write", "fork", "trim", "trim", "compact"))
            if act == "write" and len(kept[lane]) < 150:
                n = rng.randint(1, 9)
                t.grow(lane, len(kept[lane]) + n)
                for _ in range(n):
                    stamp += 1
                    row = int(t.physical_rows(torch.tensor([lane]), torch.tensor([[len(kept[lane])]]))[0, 0])
                    k[row], v[row // 16, :, :, row % 16] = stamp, -stamp
                    kept[lane].append(stamp)
            elif act == "fork" and lane != other:
                t.release(other)
                n = rng.randint(0, len(kept[lane]))
                attention.copy_blocks([k, v], *t.fork(lane, other, n))
                kept[other] = kept[lane][:n]
            elif act == "trim":
                n = rng.randint(0, len(kept[lane]))
                attention.copy_blocks([k, v], *t.trim(lane, n))
                kept[lane] = kept[lane][:n]
            elif act == "compact":
                attention.copy_blocks([k, v], *t.compact())
            _invariants(t)
            for j, want in enumerate(kept):
                rows = t.physical_rows(torch.tensor([j]), torch.arange(len(want))[None])[0]
                assert k[rows, 0, 0].tolist() == want and v[rows // 16, 0, 1, rows % 16].tolist() == [-x for x in want]


def test_model_fork_and_compact_on_the_cpu() -> None:
    """A forked slot steps as its source does; a compaction in between changes nothing."""
    import dataclasses

    cfg = dataclasses.replace(vm.tiny_cfg(), block_size=4)
    model = vm.Model(cfg, lanes=3, max_seq=32)
    ids = torch.tensor([[5, 9, 11, 3, 8, 2]])

    def step(lane, ids, base):
        lanes = model.lane_index([lane])
        model.blocks.grow(lane, base + ids.shape[1])
        res = model.forward_rows(ids, lanes, torch.tensor([base]), base + ids.shape[1])
        model.commit(res, lanes, torch.tensor([ids.shape[1]]))
        return res.hidden

    step(0, ids, 0)
    model.blocks.grow(2, 9)
    model.reset(2)
    model.fork(0, 1, 6)
    a = step(0, torch.tensor([[7, 1]]), 6)
    model.compact()
    b = step(1, torch.tensor([[7, 1]]), 6)
    assert torch.equal(a, b)
    assert not torch.equal(step(0, torch.tensor([[4]]), 8), step(1, torch.tensor([[6]]), 8))


def _slot_equal(model, a, b, length):
    return all(torch.equal(x, y) for x, y in zip(model_helpers.slot_state(model, a, length),
                                                 model_helpers.slot_state(model, b, length), strict=True))


def test_model_fork_and_compact_take_the_attached_heads_cache() -> None:
    """A fork inside a block and a compaction, with an MTP head attached: the head's rows and the next rounds'
    tokens are the source's."""
    import mtp

    model = model_helpers.build(k=2, lanes=4)
    ids = model_helpers.prompts(1, 21)[0]
    model.prefill(2, model_helpers.prompts(1, 40, seed=6)[0])  # blocks that the compaction finds free
    token = int(model.argmax(model.prefill(0, ids)[None])[0])
    model.fork(0, 1, 21)
    assert _slot_equal(model, 0, 1, 21)
    model.reset(2)
    before = [x.clone() for x in model_helpers.slot_state(model, 0, 21)]
    assert model.compact() > 0
    assert all(torch.equal(x, y) for x, y in zip(before, model_helpers.slot_state(model, 0, 21), strict=True))
    assert _slot_equal(model, 0, 1, 21)
    drafts = [mtp.draft(model, model.mtp, model.hidden_cache[[lane]], [token], [lane], [21]) for lane in (0, 1)]
    assert drafts[0] == drafts[1]
    rounds = [mtp.speculative_decode(model, [lane], [token], [21]) for lane in (0, 1)]
    assert rounds[0] == rounds[1] and _slot_equal(model, 0, 1, 21 + len(rounds[0][0]))


def test_a_head_with_a_longer_cache_than_the_layers() -> None:
    model = model_helpers.build(lanes=4)
    for name, rows in (("k", 48), ("v", 3)):
        p = model.mtp.pool[name]
        model.mtp.pool[name] = torch.cat([p, torch.full((rows, *p.shape[1:]), 7.0)])
    model.prefill(2, model_helpers.prompts(1, 40, seed=6)[0])
    model.prefill(0, model_helpers.prompts(1, 21)[0])
    model.fork(0, 1, 21)
    model.reset(2)
    before = [x.clone() for x in model_helpers.slot_state(model, 0, 21)]
    assert _slot_equal(model, 0, 1, 21) and model.compact() > 0
    assert all(torch.equal(x, y) for x, y in zip(before, model_helpers.slot_state(model, 1, 21), strict=True))
    assert bool((model.mtp.pool["k"][-48:] == 7.0).all()) and bool((model.mtp.pool["v"][-3:] == 7.0).all())


def test_caches_name_each_pool_once() -> None:
    model = model_helpers.build()
    pools = model.caches()
    assert any(p is model.mtp.pool["k"] for p in pools) and any(p is model.mtp.pool["v"] for p in pools)
    other = {"k": torch.zeros(1), "v": torch.zeros(1)}
    assert [id(p) for p in model.caches(model.mtp.pool, other)] == [id(p) for p in (*pools, other["k"], other["v"])]
    assert len({p.data_ptr() for p in pools}) == len(pools) == 2 * (1 + model.cfg.layer_types.count(vm.ATTN))


def test_a_refused_copy_leaves_the_tables_as_they_were() -> None:
    """Pools that the copy cannot take: neither a fork nor a compaction writes a table first."""
    model = model_helpers.build(lanes=3)
    model.prefill(2, model_helpers.prompts(1, 40, seed=6)[0])
    model.prefill(0, model_helpers.prompts(1, 21)[0])
    model.reset(2)
    t = model.blocks
    assert t.moves()[0]
    was = [list(h) for h in t.host], list(t.held_positions), dict(t._holders), list(t._free), t.table.clone()
    kept = [x.clone() for x in model_helpers.slot_state(model, 0, 21)]
    good = model.mtp.pool["k"], model.mtp.pool["v"]
    for bad in ({"k": good[0][:-16].clone(), "v": good[1]}, {"k": good[0][:-16].clone(), "v": good[1][:-1].clone()},
                {"k": good[0].view(-1), "v": good[1]}, {"k": good[0].transpose(1, 2), "v": good[1]}):
        for call in (lambda: model.fork(0, 1, 21, bad), lambda: model.compact(bad)):
            with pytest.raises(ValueError):
                call()
            assert (t.host, t.held_positions, t._holders, t._free) == was[:4] and torch.equal(t.table, was[4])
    short = {name: p[: p.shape[0] // 2].clone() for name, p in model.mtp.pool.items()}
    only, model.mtp = model.mtp, None
    own = model.pool
    model.pool = [short if ty == vm.ATTN else p for ty, p in zip(model.cfg.layer_types, own)]
    for call in (lambda: model.fork(0, 1, 21), lambda: model.compact()):  # pools of one number, but not the tables'
        with pytest.raises(ValueError):
            call()
        assert (t.host, t.held_positions, t._holders, t._free) == was[:4] and torch.equal(t.table, was[4])
    model.pool, model.mtp = own, only
    assert all(torch.equal(x, y) for x, y in zip(kept, model_helpers.slot_state(model, 0, 21), strict=True))
    model.fork(0, 1, 21)
    assert _slot_equal(model, 0, 1, 21) and model.compact() > 0


def test_copy_blocks_on_the_cpu_and_its_refusals() -> None:
    k, v = torch.arange(64.0).view(64, 1, 1).expand(64, 1, 4).contiguous(), torch.arange(4.0).view(4, 1, 1, 1).expand(4, 1, 4, 16).contiguous()
    attention.copy_blocks([k, v], [2, 2], [0, 3])
    assert k[:16].equal(k[32:48]) and k[48:].equal(k[32:48]) and v[:, 0, 0, 0].tolist() == [2.0, 1.0, 2.0, 2.0]
    attention.copy_blocks([k], [], [])
    before = k.clone(), v.clone()
    for pools, src, dst in (([k, v], [0], [4]), ([k, v], [-1], [1]), ([k, v], [0, 1], [2, 2]), ([k, v], [0, 1], [1, 2]),
                            ([k, v], [1], [1]), ([k, v], [0, 1], [2]), ([], [0], [1]), ([k[:40]], [0], [1]),
                            ([k, v[:3]], [0], [1]), ([k[::2]], [0], [1]), ([k.view(64, 4)], [0], [1])):
        with pytest.raises(ValueError):
            attention.copy_blocks(pools, src, dst)
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


def test_host_ids_that_are_not_integers_are_refused() -> None:
    k = torch.arange(64.0).view(64, 1, 1)
    before = k.clone()
    for src, dst in (([0.7], [1]), ([0], [1.5]), (torch.tensor([0.0]), torch.tensor([1.0])), ([True], [False]), ([0j], [1])):
        with pytest.raises(ValueError):
            attention.copy_blocks([k], src, dst)
    assert torch.equal(k, before)
    attention.copy_blocks([k], torch.tensor([2], dtype=torch.uint8), torch.tensor([[1]], dtype=torch.int32))
    attention.copy_blocks([k], [], torch.empty(0))
    assert torch.equal(k[16:32], before[32:48]) and torch.equal(k[:16], before[:16])


def test_cpu_pools_take_no_library(monkeypatch) -> None:
    """The torch spelling alone: copies, refusals, a model's fork and compaction without a built library."""
    def missing():
        raise RuntimeError("not built")

    monkeypatch.setattr(_mtpk, "native", missing)
    monkeypatch.setattr(_mtpk, "lib", missing)
    test_copy_blocks_on_the_cpu_and_its_refusals()
    test_model_fork_and_compact_take_the_attached_heads_cache()
    with pytest.raises(ValueError):
        attention.copy_blocks([torch.zeros(())], [0], [0])
    with pytest.raises(ValueError):
        attention.copy_blocks([torch.zeros(32, 1, 1)], [0], [1], 0)


def test_a_cpu_tensor_has_no_stream(monkeypatch) -> None:
    """Not the current device's either: the kernel would be handed a host address."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    for device in (torch.device("cpu"), torch.device("cpu", 0), torch.device("meta")):
        with pytest.raises(ValueError):
            _mtpk.stream_of(device)
    with pytest.raises(ValueError):
        _mtpk.stream_for(torch.empty(1))
    assert _mtpk.stream_of(torch.device("cuda")) == 0


P = 1 << 20  # an address that no refused call follows


@pytest.fixture(scope="module")
def lib():
    if not _mtpk.LIB_PATH.exists():
        import __graft_entry__

        __graft_entry__.build()
    return _mtpk.lib()


@pytest.mark.parametrize("bad", [{"pool": P + 8}, {"pool": None}, {"bytes": 24}, {"bytes": 0}, {"n": 0}, {"blocks": 0}, {"src": None},
                                 {"dst": None}, {"dt": 0}, {"pairs": -1}, {"pairs": 1 << 40}])
def test_copy_blocks_entry_point_refuses(lib, bad) -> None:
    a = {**dict(pool=P, bytes=4096, n=2, blocks=8, src=P, dst=P, dt=2, pairs=3), **bad}
    pools, sizes = (ctypes.c_void_p * 2)(P, a["pool"]), (ctypes.c_int64 * 2)(4096, a["bytes"])
    assert lib.mtpk_copy_blocks(ctypes.addressof(pools), ctypes.addressof(sizes), a["n"], a["blocks"], a["src"], a["dst"],
                                a["dt"], a["pairs"], None) == _mtpk.EINVAL


MASKED = dict(q=P, qs=(1536, 64, 512), gate=None, gs=(1536, 64, 512), b=2, t=3, heads=8, kvh=2, hd=64, kp=P, vp=P, rows=160,
              table=P, stride=5, base=P, scale=0.1, cap=0.0, window=0, slopes=None, prefix=None, pdt=0, first=None, fdt=0, n=1, ws=None,
              wsb=0, out=P, os=(1536, 64, 512))


@pytest.mark.parametrize("bad", [
    {"q": None}, {"kp": None}, {"vp": P + 4}, {"table": None}, {"base": None}, {"out": P + 2}, {"gate": P + 2}, {"b": -1}, {"t": 0},
    {"heads": 0}, {"kvh": 3}, {"kvh": 0}, {"hd": 96}, {"rows": 0}, {"rows": 150}, {"stride": 0}, {"stride": 1 << 27}, {"scale": 0.0},
    {"scale": float("nan")}, {"scale": float("inf")}, {"cap": -1.0}, {"cap": float("nan")}, {"cap": float("inf")}, {"window": -1},
    {"prefix": P, "pdt": 0}, {"first": P, "fdt": 4}, {"n": 0}, {"n": 65, "ws": P, "wsb": 1 << 30}, {"n": 2}, {"n": 2, "ws": P, "wsb": 64},
    {"n": 2, "ws": P + 4, "wsb": 1 << 30}, {"qs": (1536, 60, 512)}, {"os": (1536, 64, 511)}, {"gate": P, "gs": (1530, 64, 512)},
    {"b": 1 << 20, "t": 1 << 12},
])  # fmt: skip
def test_masked_attention_entry_point_refuses(lib, bad) -> None:
    a = {**MASKED, **bad}
    st = [(ctypes.c_int64 * 3)(*a[n]) for n in ("qs", "gs", "os")]
    qs, gs, os_ = (ctypes.addressof(s) for s in st)
    assert lib.mtpk_paged_attention_masked(
        a["q"], qs, a["gate"], gs, a["b"], a["t"], a["heads"], a["kvh"], a["hd"], a["kp"], a["vp"], a["rows"], a["table"], a["stride"],
        a["base"], a["scale"], a["cap"], a["window"], a["slopes"], a["prefix"], a["pdt"], a["first"], a["fdt"], a["n"], a["ws"], a["wsb"],
        a["out"], os_, None) == _mtpk.EINVAL


def test_masked_attention_sizes(lib) -> None:
    assert lib.mtpk_attention_masked_splits(2, 1, 8, 3, 64, 100, 0) == 0
    assert lib.mtpk_attention_masked_splits(2, 1, 8, 2, 96, 100, 0) == 0
    assert lib.mtpk_attention_masked_splits(2, 1, 8, 2, 64, 0, 0) == 1
    for ctx in (0, 100, 30000):  # a window past every context is none
        assert (lib.mtpk_attention_masked_splits(1, 1, 32, 2, 256, ctx, 2**63 - 1)
                == lib.mtpk_attention_masked_splits(1, 1, 32, 2, 256, ctx, 0))
    assert lib.mtpk_attention_masked_workspace_bytes(2, 1, 8, 2, 64, 1) == 0
    assert lib.mtpk_attention_masked_workspace_bytes(2, 1, 8, 2, 64, 3) >= 2 * 2 * 4 * 3 * 66 * 4


def test_launches_stay_within_a_grid(lib) -> None:
    """More workgroups than a launch's 2^32 threads hold: refused before the launch."""
    assert lib.mtpk_attention_masked_splits(1 << 24, 1, 1, 1, 64, 100, 0) == 0
    assert lib.mtpk_attention_masked_splits((1 << 24) - 1, 1, 1, 1, 64, 100, 0) == 1
    strides = (ctypes.c_int64 * 2)(512, 512)
    st = ctypes.addressof(strides)
    assert lib.mtpk_rotate(P, _mtpk.BF16, st, 1 << 26, 1, 512, None, 0, 1e-6, P, P, 64, 0, 1.0, P, st,
                           None) == _mtpk.EINVAL
    pools, sizes = (ctypes.c_void_p * 1)(P), (ctypes.c_int64 * 1)(1 << 40)
    assert lib.mtpk_copy_blocks(ctypes.addressof(pools), ctypes.addressof(sizes), 1, 8, P, P, 2, 3, None) == _mtpk.EINVAL


def test_a_merge_stays_within_a_grid(lib) -> None:
    """Splits that the caller chose, beyond what the sizes ask for."""
    strides = (ctypes.c_int64 * 3)(1 << 30, 64, 128)
    st = ctypes.addressof(strides)
    for n, t in ((9, 1 << 24), (64, (1 << 25) - 1)):
        size = lib.mtpk_attention_masked_workspace_bytes(1, t, 1, 1, 64, n)
        assert size > 0
        assert lib.mtpk_paged_attention_masked(P, st, None, st, 1, t, 1, 1, 64, P, P, 160, P, 5, P, 0.1, 0.0, 0, None, None, 0, None, 0, n,
                                               P, size, P, st, None) == _mtpk.EINVAL
