"""The masked attention oracle against closed forms and the plain attention oracle."""

from __future__ import annotations

import torch

from oracle import attention_ref, masked_attention_ref


def _case(seed, b=2, t=5, heads=4, kvh=2, hd=8, base=(9, 20), blocks=3):
    g = torch.Generator().manual_seed(seed)
    n = b * blocks + 1
    table = (torch.randperm(n - 1, generator=g) + 1).view(b, blocks)
    q = torch.randn(b, t, heads, hd, generator=g, dtype=torch.float64)
    k, v = (torch.randn(n * 16, kvh, hd, generator=g, dtype=torch.float64) for _ in range(2))
    return q, k, v, table, torch.tensor(base)


def _values(v, table, i, j, kv):
    return v[table[i][j // 16] * 16 + j % 16, kv]


def test_plain_is_causal_attention() -> None:
    q, k, v, table, base = _case(0)
    out, spread = masked_attention_ref.paged_attention_masked(q, k, v, table, base, 0.3)
    want = attention_ref.paged_attention(q.transpose(1, 2), k, v, table.numpy(), base.numpy(), 0.3)
    torch.testing.assert_close(out.transpose(1, 2), torch.from_numpy(want), rtol=1e-12, atol=1e-13)
    assert torch.all(spread >= out.abs() - 1e-12)
    far, _ = masked_attention_ref.paged_attention_masked(q, k, v, table, base, 0.3, softcap=1e7)
    torch.testing.assert_close(far, out, rtol=1e-9, atol=1e-10)


def test_masks_admit_what_they_say() -> None:
    """Identical keys: a row is the mean of the values that it sees."""
    q, k, v, table, base = _case(1)
    k = k[:1].expand_as(k)
    prefix, first = torch.tensor([12, 3]), torch.tensor([[0, 5, 11, 30, 9], [7, 21, 22, 23, 2]])
    for kw in ({}, {"window": 3}, {"prefix": prefix}, {"first": first}, {"window": 6, "prefix": prefix, "first": first}):
        out, _ = masked_attention_ref.paged_attention_masked(q, k, v, table, base, 0.5, **kw)
        for i in range(2):
            for s in range(5):
                p = int(base[i]) + s
                keys = [j for j in range(int(base[i]) + 5)
                        if (j <= p or ("prefix" in kw and p < prefix[i] and j < prefix[i]))
                        and ("window" not in kw or p - j < kw["window"]) and ("first" not in kw or j >= first[i, s])]
                want = _values(v, table, i, torch.tensor(keys), 1).mean(0) if keys else torch.zeros(8, dtype=torch.float64)
                torch.testing.assert_close(out[i, s, 3], want, rtol=1e-11, atol=1e-12)


def test_caps_and_slopes() -> None:
    q, k, v, table, base = _case(2)
    out, _ = masked_attention_ref.paged_attention_masked(q, k, v, table, base, 5.0, softcap=1e-9)
    torch.testing.assert_close(out[1, 2, 0], _values(v, table, 1, torch.arange(23), 0).mean(0), rtol=1e-7, atol=1e-8)
    slopes = torch.tensor([0.0, 1e4, 0.0, 1e4])
    out, _ = masked_attention_ref.paged_attention_masked(q, k, v, table, base, 0.3, slopes=slopes)
    torch.testing.assert_close(out[0, 4, 3], _values(v, table, 0, torch.tensor([13]), 1)[0], rtol=1e-12, atol=0)


def test_unseen_values_stay_out() -> None:
    q, k, v, table, base = _case(3)
    clean, _ = masked_attention_ref.paged_attention_masked(q, k, v, table, base, 0.3)
    v[table[0][0] * 16 + 11] = float("nan")  # position 11 of lane 0: rows 2.. see it
    out, _ = masked_attention_ref.paged_attention_masked(q, k, v, table, base, 0.3)
    assert torch.equal(out[0, :2], clean[0, :2]) and out[0, 2:].isnan().all() and torch.equal(out[1], clean[1])


def test_a_bias_goes_by_the_distances_differences() -> None:
    """A row far behind its keys weighs them as the nearest row that sees them all: one distance more for every key
    is no change, to the digits of 64 bits."""
    q, k, v, table, _ = _case(3, b=1, t=1, base=(0,))
    slopes = torch.tensor([0.01, 0.1, 0.3, 1.0])
    near, _ = masked_attention_ref.paged_attention_masked(q, k, v, table, torch.tensor([48]), 0.5, slopes=slopes)
    for past in (1, 2**20, 2**31):
        far, _ = masked_attention_ref.paged_attention_masked(q, k, v, table, torch.tensor([48 + past]), 0.5, slopes=slopes)
        torch.testing.assert_close(far, near, rtol=1e-6, atol=1e-7)
