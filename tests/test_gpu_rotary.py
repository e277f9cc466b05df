"""Head rotation (`mtpk_rotate`) and the rows' way into the cache (`mtpk_rotate_to_cache`) against a 64-bit
restatement. Bars: one rounding to the output type (at most half a step, 2^-8 of the value in bf16, 2^-24
in fp32) and the fp32 arithmetic before it: norm, cosine and sine and the pair's two products, each a few
roundings of 2^-24 of the pair's length, 16 of them (2^-20) allowed."""

from __future__ import annotations

import pytest
import torch

import attention
import rotary
import verify_model as vm

pytestmark = pytest.mark.gpu


def exact(x, pos, rates, magnitude, interleaved, w, eps):
    """64 bits on the CPU; also the length of each channel's pair (of the channel itself past the pairs)."""
    y = x.double().cpu()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (1 + w.double().cpu())
    half, rates = rates.shape[0], rates.cpu()
    at = torch.arange(half)
    i, j = (2 * at, 2 * at + 1) if interleaved else (at, at + half)
    ang = (pos.double().cpu()[..., None] * rates)[..., None, :]
    out, size = y.clone(), y.abs()
    a, b = y[..., i], y[..., j]
    out[..., i] = (a * ang.cos() - b * ang.sin()) * magnitude
    out[..., j] = (b * ang.cos() + a * ang.sin()) * magnitude
    size[..., i] = size[..., j] = torch.hypot(a, b) * magnitude
    return out, size


def close(got, want, size):
    step = torch.finfo(got.dtype).eps / 2
    off = (got.double().cpu() - want).abs()
    bar = step * want.abs() + 2.0**-20 * size
    assert torch.all(off <= bar), float((off / bar.clamp_min(1e-300)).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,rot,interleaved,norm", [
    (1, 1, 8, 2, False, True),
    (1, 32, 256, 64, False, True),
    (48, 32, 256, 64, False, True),
    (5, 3, 16, 16, True, False),
    (7, 5, 80, 40, False, True),       # halves of 20: pairs across the lanes' eights
    (7, 5, 96, 96, True, True),
    (3, 2, 192, 128, False, False),
    (130, 9, 512, 510, False, True),
    (130, 9, 512, 512, True, True),
    (4, 17, 64, 6, False, True),
    (2051, 11, 128, 128, False, True),  # one workgroup a token
    (4100, 2, 40, 24, True, False),
])  # fmt: skip
def test_rotate(dev, dtype, tokens, heads, dim, rot, interleaved, norm) -> None:
    g = torch.Generator(dev).manual_seed(tokens + dim)
    x = (torch.randn(tokens, heads, dim, device=dev, generator=g) * 3).to(dtype)
    w = (torch.randn(dim, device=dev, generator=g) * 0.3).to(dtype) if norm else None
    pos = torch.randint(0, 1 << 20, (tokens,), device=dev, generator=g)
    rates, m = rotary.frequencies(rot, 1e6, scaling="yarn", factor=4.0, original=4096, device=dev)
    got = rotary.rotate(x, pos, rates, magnitude=m, interleaved=interleaved, w=w, eps=1e-5)
    assert got.dtype == dtype and got.shape == x.shape
    close(got, *exact(x, pos, rates, m, interleaved, w, 1e-5))
    again = rotary.rotate(x, pos, rates, magnitude=m, interleaved=interleaved, w=w, eps=1e-5, out=x)
    assert again is x and torch.equal(x, got)  # in place


def test_far_and_negative_positions(dev) -> None:
    """The angle of a position past 2^31, and of one before 0, to fp32's last bits."""
    x = torch.randn(4, 2, 64, device=dev)
    pos = torch.tensor([2**33 + 12345, -7, 0, 2**31 - 1], device=dev)
    rates, _ = rotary.frequencies(64, 1e4, device=dev)
    got = rotary.rotate(x, pos, rates)
    want, size = exact(x, pos, rates, 1.0, False, None, 0.0)
    # position * rate in 64 bits is itself off by 2^-53 of 1.4e9 turns, 2e-7 of a turn, on either side
    assert float(((got.double().cpu() - want).abs() / size)[0].max()) < 2e-6
    close(got[1:], want[1:], size[1:])
    assert torch.equal(got[2], x[2])


def test_strides_and_types(dev) -> None:
    """Head slices in place, rows off 16 bytes (copied), transposed heads, a wide output row, fp32
    weights of bf16 heads, 32-bit positions, and what is not finite staying in its head."""
    g = torch.Generator(dev).manual_seed(0)
    rates, m = rotary.frequencies(32, 1e4, device=dev)
    full = torch.randn(3, 5, 4, 131, device=dev, generator=g).bfloat16()
    pos = torch.arange(15, device=dev, dtype=torch.int32).view(3, 5)
    w = torch.randn(64, device=dev, generator=g) * 0.1
    for x in (full[..., 64:128], full[..., 1:65], full[..., :64].transpose(0, 1).contiguous().transpose(0, 1),
              full[:, :, :, :64].transpose(1, 2).contiguous().transpose(1, 2)):
        close(rotary.rotate(x, pos, rates, w=w), *exact(x, pos, rates, m, False, w, 1e-6))
    x = full[..., :64].contiguous()
    wide = torch.zeros(3, 5, 4, 128, device=dev, dtype=torch.bfloat16)
    rotary.rotate(x, pos, rates, w=w, out=wide[..., 64:])
    close(wide[..., 64:], *exact(x, pos, rates, m, False, w, 1e-6))
    assert not wide[..., :64].any()
    x[1, 2, 3, 40] = float("inf")  # past the pairs: its head alone, and without a norm itself alone
    got, clean = rotary.rotate(x, pos, rates), rotary.rotate(x.nan_to_num(posinf=0.0), pos, rates)
    off = got != clean
    assert int(off.sum()) == 1 and bool(off[1, 2, 3, 40])


def test_another_stream_and_a_graph(dev) -> None:
    rates, m = rotary.frequencies(64, 1e4, device=dev)
    x = torch.randn(9, 4, 128, device=dev).bfloat16()
    pos = torch.arange(9, device=dev)
    want = rotary.rotate(x, pos, rates)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotary.rotate(x, pos, rates)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rotary.rotate(x, pos, rates)
    for i in range(4):
        x.copy_(torch.randn_like(x))
        pos.add_(100 * i)
        graph.replay()
        assert torch.equal(got, rotary.rotate(x, pos, rates))


def test_rotate_refuses(dev) -> None:
    rates, _ = rotary.frequencies(64, 1e4, device=dev)
    x, pos = torch.randn(4, 2, 64, device=dev), torch.arange(4, device=dev)
    for bad in (lambda: rotary.rotate(x, pos[:3], rates), lambda: rotary.rotate(x, pos.float(), rates),
                lambda: rotary.rotate(x.half(), pos, rates), lambda: rotary.rotate(x, pos, rates.float()),
                lambda: rotary.rotate(x[..., :32], pos, rates), lambda: rotary.rotate(x.cpu(), pos, rates),
                lambda: rotary.rotate(x, pos, rates, w=x[0, 0, :32]), lambda: rotary.rotate(x, pos, rates, out=x[:3]),
                lambda: rotary.rotate(torch.randn(4, 2, 68, device=dev), pos, rates)):
        with pytest.raises(ValueError):
            bad()
    assert rotary.rotate(x[:0], pos[:0], rates).shape == (0, 2, 64)


def _round(dev, b, t, heads, kvh, hd, rot, base, seed, blocks):
    g = torch.Generator(dev).manual_seed(seed)
    n = b * blocks + 1
    table = (torch.randperm(n - 1, device=dev, generator=g) + 1).view(b, blocks).int()
    qkv = torch.randn(b, t, (2 * heads + 2 * kvh) * hd, device=dev, generator=g).bfloat16() * 2
    q = qkv[..., : 2 * heads * hd].view(b, t, heads, 2 * hd)[..., :hd]
    k, v = (qkv[..., (2 * heads + i * kvh) * hd :][..., : kvh * hd].view(b, t, kvh, hd) for i in range(2))
    pools = torch.randn(n * 16, kvh, hd, device=dev, generator=g).bfloat16(), torch.randn(n, kvh, hd, 16, device=dev, generator=g).bfloat16()
    return q, k, v, pools, table, torch.tensor(base, device=dev)


@pytest.mark.parametrize("b,t,heads,kvh,hd,rot,interleaved,base", [
    (1, 1, 32, 2, 256, 64, False, [0]),
    (4, 4, 32, 2, 256, 64, False, [0, 13, 15, 700]),
    (3, 5, 8, 2, 64, 64, True, [11, 12, 31]),
    (2, 37, 16, 4, 128, 20, False, [3, 16]),
    (1, 300, 6, 3, 48, 48, True, [5]),
    (1, 2100, 4, 1, 256, 256, False, [0]),
    (2, 1, 1, 1, 512, 128, False, [1, 14]),
])  # fmt: skip
def test_rotate_to_cache(dev, b, t, heads, kvh, hd, rot, interleaved, base) -> None:
    q, k, v, (kp, vp), table, pos0 = _round(dev, b, t, heads, kvh, hd, rot, base, t + hd, (max(base) + t) // 16 + 2)
    rates, m = rotary.frequencies(rot, 1e6, scaling="linear", factor=2.0, device=dev)
    qn, kn = (torch.randn(hd, device=dev).bfloat16() * 0.2 for _ in range(2))
    keep = torch.rand(b, t, device=dev) < 0.8
    kp0, vp0 = kp.clone(), vp.clone()
    got = rotary.rotate_to_cache(q, k, v, rates, kp, vp, table, pos0, magnitude=0.75, interleaved=interleaved,
                                 q_norm=qn, k_norm=kn, keep=keep)
    pos = pos0[:, None] + torch.arange(t, device=dev)
    close(got, *exact(q, pos, rates, 0.75, interleaved, qn, 1e-6))
    want, size = exact(k, pos, rates, 0.75, interleaved, kn, 1e-6)
    rows = vm.table_rows(table, pos, 16)
    close(kp[rows][keep], want[keep.cpu()], size[keep.cpu()])
    assert torch.equal(attention.read_v(vp, rows)[keep], v[keep])
    # and nothing else: rows that are not kept, other slots, other blocks
    kp0[rows[keep]] = kp[rows[keep]]
    attention.write_v(vp0, rows[keep], v[keep])
    assert torch.equal(kp, kp0) and torch.equal(vp, vp0)
    # the same values as the kernel of the heads alone
    assert torch.equal(got, rotary.rotate(q, pos, rates, magnitude=0.75, interleaved=interleaved, w=qn))


def test_rotate_to_cache_as_the_separate_calls(dev) -> None:
    """q, k and the cache of rownorm + kv_write, up to their rounding of the norm before the rotation."""
    q, k, v, (kp, vp), table, pos0 = _round(dev, 3, 4, 32, 2, 256, 64, [0, 90, 200], 3, 14)
    cfg = vm.verify_cfg()
    rates, _ = rotary.frequencies(64, cfg.rope_theta, device=dev)
    cos, sin = vm.rope_table(cfg, 256, dev)
    qn, kn = (torch.randn(256, device=dev).bfloat16() * 0.2 for _ in range(2))
    pos = (pos0[:, None] + torch.arange(4, device=dev)).reshape(-1)
    import rownorm

    q2, k2 = (rownorm.rmsnorm(x, w, 1e-6, heads=True, rope=(cos, sin, pos)) for x, w in ((q, qn), (k, kn)))
    kp2, vp2 = kp.clone(), vp.clone()
    attention.kv_write(kp2, vp2, k2, v, table, pos0)
    got = rotary.rotate_to_cache(q, k, v, rates, kp, vp, table, pos0, q_norm=qn, k_norm=kn)
    # the norm's rounding is half a step of either value of the pair, then the output's own, on each side;
    # the fp32 table's angle is off by 2^-24 of up to 204 radians
    for a, b in ((got, q2), (kp, kp2)):
        size = a.float().abs() + torch.cat([a.float()[..., 32:64], a.float()[..., :32], a.float()[..., 64:]], -1).abs()
        assert torch.all((a.float() - b.float()).abs() <= (3 * 2.0**-8 + 1e-4) * size)
    assert torch.equal(vp, vp2)


def test_cache_rows_outside_the_table_or_pool(dev) -> None:
    q, k, v, (kp, vp), table, _ = _round(dev, 4, 2, 4, 2, 64, 64, [0] * 4, 1, 3)
    rates, _ = rotary.frequencies(64, 1e4, device=dev)
    table[2, 0], table[3, 0] = -1, 10**6
    base = torch.tensor([-1, 3 * 16 - 1, 0, 5], device=dev)  # before the table; past its end; no such block
    kp0, vp0 = kp.clone(), vp.clone()
    got = rotary.rotate_to_cache(q, k, v, rates, kp, vp, table, base)
    pos = base[:, None] + torch.arange(2, device=dev)
    close(got, *exact(q, pos, rates, 1.0, False, None, 0.0))
    want, size = exact(k, pos, rates, 1.0, False, None, 0.0)
    live = [(0, 1, int(table[0, 0]) * 16), (1, 0, int(table[1, 2]) * 16 + 15)]
    for b, s, row in live:
        close(kp[row], want[b, s], size[b, s])
        assert torch.equal(vp[row // 16, :, :, row % 16], v[b, s])
        kp0[row], vp0[row // 16, :, :, row % 16] = kp[row], v[b, s]
    assert torch.equal(kp, kp0) and torch.equal(vp, vp0)


def test_cache_in_a_graph_with_positions_of_its_own(dev) -> None:
    q, k, v, (kp, vp), table, base = _round(dev, 2, 3, 8, 2, 128, 128, [4, 30], 5, 6)
    rates, _ = rotary.frequencies(128, 1e4, device=dev)
    at = torch.randint(0, 1000, (2, 3), device=dev)
    keep = torch.ones(2, 3, dtype=torch.bool, device=dev)
    args = (q, k, v, rates, kp, vp, table, base)
    rotary.rotate_to_cache(*args, positions=at, keep=keep)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rotary.rotate_to_cache(*args, positions=at, keep=keep)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        k.copy_(torch.randn_like(k))
        base.add_(1)
        keep[i % 2, i % 3] = not bool(keep[i % 2, i % 3])
        kp2, vp2 = kp.clone(), vp.clone()
        graph.replay()
        want = rotary.rotate_to_cache(q, k, v, rates, kp2, vp2, table, base, positions=at, keep=keep)
        assert torch.equal(got, want) and torch.equal(kp, kp2) and torch.equal(vp, vp2)
        close(got, *exact(q, at, rates, 1.0, False, None, 0.0))


def test_rotate_to_cache_refuses(dev) -> None:
    q, k, v, (kp, vp), table, base = _round(dev, 2, 3, 8, 2, 64, 64, [4, 30], 5, 6)
    rates, _ = rotary.frequencies(64, 1e4, device=dev)

    def call(**kw):
        a = dict(q=q, k=k, v=v, rates=rates, k_pool=kp, v_pool=vp, block_table=table, base_pos=base)
        rest = {n: x for n, x in kw.items() if n not in a}
        rotary.rotate_to_cache(*{**a, **{n: x for n, x in kw.items() if n in a}}.values(), **rest)

    before = kp.clone(), vp.clone()
    for kw in ({"q": q.float()}, {"k": k[:, :2]}, {"v": v[..., :32]}, {"k_pool": kp[:8]}, {"v_pool": vp[:-1]},
               {"v_pool": vp.transpose(2, 3)}, {"block_table": table[:1]}, {"block_table": table.float()},
               {"base_pos": base[:1]}, {"rates": rates.float()}, {"k": k[:, :, :1], "v": v[:, :, :1]},
               {"keep": torch.ones(2, 3, device=dev)}, {"keep": torch.ones(2, 3, device=dev, dtype=torch.int8)},
               {"keep": torch.ones(3, 2, dtype=torch.bool, device=dev)},
               {"positions": torch.zeros(2, 3, device=dev)}, {"q_norm": torch.zeros(32, device=dev)},
               {"q_norm": torch.zeros(64, device=dev), "k_norm": torch.zeros(64, device=dev).bfloat16()}):
        with pytest.raises(ValueError):
            call(**kw)
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])


def test_rotate_to_cache_of_no_rows_and_of_no_heads(dev) -> None:
    """No rows are no work; k and v beside a q without heads are not left unwritten in silence."""
    q, k, v, (kp, vp), table, base = _round(dev, 2, 3, 8, 2, 64, 64, [4, 30], 5, 6)
    rates, _ = rotary.frequencies(64, 1e4, device=dev)
    before = kp.clone(), vp.clone()
    assert rotary.rotate_to_cache(q[:, :0], k[:, :0], v[:, :0], rates, kp, vp, table, base).shape == (2, 0, 8, 64)
    assert rotary.rotate_to_cache(q[:0], k[:0], v[:0], rates, kp, vp, table[:0], base[:0]).shape == (0, 3, 8, 64)
    with pytest.raises(ValueError):
        rotary.rotate_to_cache(q[:, :, :0], k, v, rates, kp, vp, table, base)
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])
