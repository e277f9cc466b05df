"""Block copies on the device (`mtpk_copy_blocks`) against indexing, bit for bit, and a model's fork and
compaction."""

from __future__ import annotations

import pytest
import torch

import _mtpk
import attention
import verify_model as vm
from tests import model_helpers

pytestmark = pytest.mark.gpu


def _pools(dev, layers, blocks, kvh, hd, dtype=torch.bfloat16):
    g = torch.Generator(dev).manual_seed(blocks)
    k = [torch.randn(blocks * 16, kvh, hd, device=dev, generator=g).to(dtype) for _ in range(layers)]
    v = [torch.randn(blocks, kvh, hd, 16, device=dev, generator=g).to(dtype) for _ in range(layers)]
    return k + v


def _want(pools, src, dst, blocks):
    out = []
    for p in pools:
        x = p.clone().view(blocks, -1)
        x[dst.long()] = p.view(blocks, -1)[src.long()]
        out.append(x.view(p.shape))
    return out


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("layers,blocks,kvh,hd,pairs,dtype", [
    (1, 2, 1, 8, 1, torch.bfloat16),       # 256-byte blocks
    (15, 40, 2, 256, 3, torch.bfloat16),
    (40, 50, 1, 24, 20, torch.float32),    # 80 pools: two launches
    (2, 700, 4, 128, 349, torch.bfloat16),
    (1, 64, 5, 256, 30, torch.float32),    # blocks of several pieces, the last one partial
])  # fmt: skip
def test_copies(dev, layers, blocks, kvh, hd, pairs, dtype, index) -> None:
    pools = _pools(dev, layers, blocks, kvh, hd, dtype)
    order = torch.randperm(blocks, device=dev).to(index)
    src, dst = order[:pairs], order[pairs : 2 * pairs]
    src = src[torch.randint(0, pairs, (pairs,), device=dev)]  # a block may be copied several times
    want = _want(pools, src, dst, blocks)
    attention.copy_blocks(pools, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    attention.copy_blocks(pools, src.tolist(), dst.tolist())  # checked lists, the same copies again
    attention.copy_blocks(pools, src.cpu(), dst.cpu())
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_ids_outside_the_pools_are_skipped(dev) -> None:
    pools = _pools(dev, 1, 9, 2, 64)
    src = torch.tensor([-1, 3, 9, 4, 5], device=dev)
    dst = torch.tensor([2, -7, 1, 2**40, 0], device=dev)
    want = _want(pools, src[4:], dst[4:], 9)
    attention.copy_blocks(pools, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_in_a_graph(dev) -> None:
    pools = _pools(dev, 2, 30, 2, 128)
    src, dst = torch.tensor([3, 4], device=dev), torch.tensor([10, 11], device=dev)
    attention.copy_blocks(pools, src, dst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention.copy_blocks(pools, src, dst)
    for i in range(4):
        src.add_(1)
        dst.add_(2)
        for p in pools:
            p.add_(1.0)
        want = _want(pools, src, dst, 30)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_host_ids_are_refused_in_a_capture(dev) -> None:
    """The graph would read the host's ids again at every replay, long after they are gone."""
    pools = _pools(dev, 1, 8, 2, 64)
    attention.copy_blocks(pools, [1], [2])
    before = [p.clone() for p in pools]
    src, dst = torch.tensor([3], device=dev), torch.tensor([4], device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention.copy_blocks(pools, src, dst)
        with pytest.raises(ValueError, match="graph"):
            attention.copy_blocks(pools, [1], [5])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(pools, _want(before, src, dst, 8)))


def test_stream_handles(dev) -> None:
    """The current stream's handle, of a device with and without an index."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for device in (torch.device("cuda"), torch.device("cuda", torch.cuda.current_device())):
            assert _mtpk.stream_of(device) == stream.cuda_stream
        assert _mtpk.stream_for(torch.empty(1, device=dev)) == stream.cuda_stream


def test_offsets_past_four_gigabytes(dev) -> None:
    kvh, hd = 8, 256
    blocks = 2**32 // (16 * kvh * hd * 2) + 64
    k = torch.empty(blocks * 16, kvh, hd, dtype=torch.bfloat16, device=dev)
    a, b = blocks - 1, 3
    k[a * 16 : a * 16 + 16] = torch.randn(16, kvh, hd, device=dev).bfloat16()
    k[40 * 16 : 41 * 16] = 7.0
    attention.copy_blocks([k], [a, 40], [b, blocks - 2])
    assert torch.equal(k[b * 16 : b * 16 + 16], k[a * 16 :]) and bool((k[(blocks - 2) * 16 : (blocks - 1) * 16] == 7.0).all())


def test_refusals(dev) -> None:
    pools = _pools(dev, 1, 8, 2, 64)
    before = [p.clone() for p in pools]
    i = torch.tensor([1], device=dev)
    for call in (lambda: attention.copy_blocks(pools, [1, 2], [3, 3]), lambda: attention.copy_blocks(pools, [8], [0]),
                 lambda: attention.copy_blocks(pools, i, [2]), lambda: attention.copy_blocks(pools, i, i.int()),
                 lambda: attention.copy_blocks(pools, i.float(), i.float()), lambda: attention.copy_blocks([pools[0].cpu(), pools[1]], [1], [2]),
                 lambda: attention.copy_blocks([torch.zeros(40, dtype=torch.uint8, device=dev)[8:].view(32, 1, 1)], [1], [0])):
        with pytest.raises(ValueError):
            call()
    assert all(torch.equal(a, b) for a, b in zip(pools, before))


def test_a_forked_slot_steps_as_its_source(dev) -> None:
    cfg = vm.tiny_cfg()
    model = vm.Model(cfg, device=dev, dtype=torch.float32, lanes=3, max_seq=64)

    def step(lane, ids, base):
        ids, lanes = torch.tensor([ids], device=dev), model.lane_index([lane])
        model.blocks.grow(lane, base + ids.shape[1])
        res = model.forward_rows(ids, lanes, torch.tensor([base], device=dev), base + ids.shape[1])
        model.commit(res, lanes, torch.tensor([ids.shape[1]], device=dev))
        return res.hidden

    step(0, list(range(2, 23)), 0)
    model.fork(0, 2, 21)
    a = step(0, [7, 1], 21)
    assert model.compact() > 0
    assert torch.equal(step(2, [7, 1], 21), a)
    assert not torch.equal(step(0, [4], 23), step(2, [6], 23))


def test_a_forked_slot_takes_the_attached_heads_cache(dev) -> None:
    """A fork inside a block and a compaction, with an MTP head attached: its rows and the next round's tokens
    are the source's."""
    import mtp

    model = model_helpers.build(dev, k=2, lanes=4)
    token = int(model.argmax(model.prefill(0, model_helpers.prompts(1, 21)[0])[None])[0])
    model.prefill(2, model_helpers.prompts(1, 40, seed=6)[0])
    model.fork(0, 1, 21)
    model.reset(2)
    before = [x.clone() for x in model_helpers.slot_state(model, 0, 21)]
    assert model.compact() > 0
    for lane in (0, 1):
        assert all(torch.equal(x, y) for x, y in zip(before, model_helpers.slot_state(model, lane, 21), strict=True))
    rounds = [mtp.speculative_decode(model, [lane], [token], [21]) for lane in (0, 1)]
    assert rounds[0] == rounds[1]


def test_a_fork_or_compaction_in_a_capture_changes_no_table(dev) -> None:
    model = vm.Model(vm.tiny_cfg(), device=dev, dtype=torch.float32, lanes=3, max_seq=64)
    model.blocks.grow(1, 40)
    model.blocks.grow(0, 21)
    model.reset(1)
    t = model.blocks
    was = [list(h) for h in t.host], list(t._free), t.table.clone()
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=dev)
    with torch.cuda.graph(graph):
        x.add_(1)
        for call in (lambda: model.fork(0, 2, 21), lambda: model.compact()):
            with pytest.raises(ValueError):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert (t.host, t._free) == was[:2] and torch.equal(t.table, was[2])
    model.fork(0, 2, 21)
    assert model.compact() > 0


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_more_pieces_than_a_launch_takes(dev, dtype) -> None:
    """Blocks of 16 bytes in 64 pools and two more, 2^24 pieces and some: the copies go on in a second launch."""
    n, pairs = 540000, 2**18 + 77
    pools = [torch.randint(0, 2**40, (n, 1, 2), device=dev).view(torch.int64) for _ in range(66)]
    order = torch.randperm(n, device=dev).to(dtype)
    src, dst = order[:pairs].contiguous(), order[pairs : 2 * pairs].contiguous()
    src[5], dst[pairs - 3] = -1, n  # skipped
    live = torch.ones(pairs, dtype=torch.bool, device=dev)
    live[5] = live[pairs - 3] = False
    want = []
    for p in (pools[0], pools[40], pools[63], pools[64], pools[65]):
        w = p.clone()
        w[dst[live].long()] = p[src[live].long()]
        want.append(w)
    attention.copy_blocks(pools, src, dst, 1)
    for p, w in zip((pools[0], pools[40], pools[63], pools[64], pools[65]), want, strict=True):
        assert torch.equal(p, w)
