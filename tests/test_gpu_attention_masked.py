"""Masked paged attention against its 64-bit oracle.

Bars, value by value. A probability is rounded to bf16 (half a step: 2^-8 of it) and the row's sum adds
the rounded ones, so the output is off by at most 2^-8 sum_j w_j |v_j - out| <= 2^-8 (spread + |out|), with
spread = sum_j w_j |v_j|; its own rounding adds 2^-8 |out|. The fp32 scores behind the probabilities: a sum of
up to 256 products (2^-16 of sum |q k| scale, a few units), cap and bias of up to some hundred units in
log2 at 2^-23 each, and the exponential: 3e-4 of a weight is allowed, twice for the row's sum."""

from __future__ import annotations

import math
import random

import pytest
import torch

import attention
from oracle import masked_attention_ref as ref

pytestmark = pytest.mark.gpu


def bars(want, spread):
    return 2.0**-8 * (spread + 2 * want.abs()) * (1 + 2.0**-7) + 6e-4 * spread + 1e-30


def case(seed, b, t, heads, kvh, hd, base, *, spare=1, q_std=1.0):
    g = torch.Generator().manual_seed(seed)
    blocks = max((max(base) + t + 15) // 16 + spare, 1)
    n = b * blocks + 1
    table = (torch.randperm(n - 1, generator=g) + 1).view(b, blocks).int()
    q = (torch.randn(b, t, heads, hd, generator=g) * q_std).bfloat16()
    k, v = (torch.randn(n * 16, kvh, hd, generator=g).bfloat16() for _ in range(2))
    return q, k, v, table, torch.tensor(base)


def run(dev, q, k, v, table, base, scale, ctx=None, **kw):
    kw = {n: x.to(dev) if torch.is_tensor(x) else x for n, x in kw.items()}
    ctx = max(int(base.max()) + q.shape[1], 0) if ctx is None else ctx
    return attention.paged_attention_masked(q.to(dev), k.to(dev), attention.v_blocks(v).to(dev), table.to(dev), base.to(dev),
                                            ctx, scale, **kw)


def check(dev, q, k, v, table, base, scale, **kw):
    got = run(dev, q, k, v, table, base, scale, **kw).double().cpu()
    want, spread = ref.paged_attention_masked(q, k, v, table, base, scale, **kw)
    off = (got - want).abs()
    assert not bool(got.isnan().any())
    worst = float((off / bars(want, spread)).max())
    assert worst <= 1.0
    return got


SHAPES = [  # heads, kv heads, hd, t, base
    (8, 2, 64, 1, [0]),                  # one key
    (8, 2, 64, 1, [299, 15, 16, 31]),
    (32, 2, 256, 1, [700, 0, 33]),       # one wave of 16 rows
    (16, 4, 128, 1, [5000, 77]),         # key splits, one lane's mostly empty
    (32, 2, 256, 2, [40, 95]),           # 32 rows
    (6, 2, 128, 5, [30]),                # 15 rows, odd group
    (32, 2, 256, 4, [600, 0, 13]),       # 64 rows: two waves
    (16, 4, 128, 9, [250]),              # 36 rows
    (8, 2, 64, 16, [3, 64]),             # exactly two waves
    (32, 2, 256, 5, [1000, 7]),          # 80 rows: four waves, the last two with repeats
    (32, 2, 256, 8, [0]),                # exactly four waves
    (32, 2, 256, 9, [23, 500]),          # one row past them
    (6, 2, 128, 50, [3]),                # a group that does not divide 32
    (16, 4, 128, 33, [0, 700]),
    (4, 4, 64, 200, [0]),                # no grouping
    (8, 2, 64, 65, [64]),
    (5, 1, 64, 150, [100]),
]  # fmt: skip


def masks(kind, t, heads, base, seed):
    g = torch.Generator().manual_seed(seed + 99)
    b = len(base)
    slopes = (2.0 ** (-8.0 * (1 + torch.arange(heads)) / heads)).float()
    pos = torch.tensor(base)[:, None] + torch.arange(t)
    return {
        "plain": {},
        "cap": {"softcap": 30.0},
        "window": {"window": 37, "softcap": 50.0},
        "window1": {"window": 1},
        "slopes": {"slopes": slopes},
        "documents": {"first": (pos - pos % 29).int(), "softcap": 20.0},
        "prefix": {"prefix": torch.tensor(base) + (t + 1) // 2},
        "all": {"softcap": 15.0, "window": 45, "slopes": slopes, "prefix": (torch.tensor(base) + t).int(),
                "first": pos - pos % 41, "gate": torch.randn(b, t, heads, 1, generator=g)},
        # rows that see nothing among rows that do; documents in no order
        "empty": {"first": torch.where(torch.rand(b, t, generator=g) < 0.4, pos + 1, torch.randint(0, 50, (b, t), generator=g))},
    }[kind]  # fmt: skip


@pytest.mark.parametrize("kind", ["plain", "cap", "window", "window1", "slopes", "documents", "prefix", "all", "empty"])
@pytest.mark.parametrize("heads,kvh,hd,t,base", SHAPES)
def test_against_the_oracle(dev, heads, kvh, hd, t, base, kind) -> None:
    q, k, v, table, b0 = case(t + hd, len(base), t, heads, kvh, hd, base)
    kw = masks(kind, t, heads, base, t)
    if "gate" in kw:
        kw["gate"] = (kw["gate"] + torch.zeros(hd)).bfloat16()
    got = check(dev, q, k, v, table, b0, hd**-0.5, **kw)
    if kind == "empty":
        pos = b0[:, None] + torch.arange(t)
        none = kw["first"] > pos
        assert not got[none].any()


@pytest.mark.parametrize("seed", range(16))
def test_any_mix(dev, seed) -> None:
    """Sizes, groups and masks drawn together."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    hd, kvh, group = (64, 128, 256)[seed % 3], rng.choice([1, 2, 3, 5]), rng.choice([1, 2, 3, 5, 8, 16, 33, 64])
    heads, b = kvh * group, rng.choice([1, 2, 3])
    t = max(1, min(rng.choice([1, 2, 5, 17, 64, 257]), 4000 // (heads * b)))
    base = [rng.choice([0, 15, 16, 33, rng.randrange(2000)]) for _ in range(b)]
    q, k, v, table, b0 = case(seed, b, t, heads, kvh, hd, base)
    pos = b0[:, None] + torch.arange(t)
    mixed = {"softcap": rng.choice([5.0, 50.0, 80.0]), "window": rng.choice([1, 31, 33, 64, 1000]),
             "slopes": torch.rand(heads, generator=g) * rng.choice([0.1, 1.0, -0.05]),
             "prefix": b0 + torch.randint(-3, t + 3, (b,), generator=g),
             "first": (pos - torch.randint(-2, 80, (b, t), generator=g)).int(),
             "gate": torch.randn(b, t, heads, hd, generator=g).bfloat16()}  # fmt: skip
    check(dev, q, k, v, table, b0, hd**-0.5, **{n: x for n, x in mixed.items() if rng.random() < 0.5})


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(32, 2, 256, 1, [500]), (32, 2, 256, 40, [9]), (16, 4, 128, 12, [90])])
def test_scores_past_the_polynomial(dev, heads, kvh, hd, t, base) -> None:
    """Scores of the cap's size and far above it: the cap's own bends, not its line through zero."""
    q, k, v, table, b0 = case(1, 1, t, heads, kvh, hd, base, q_std=8.0)
    check(dev, q, k, v, table, b0, hd**-0.5, softcap=2.0)
    check(dev, q, k, v, table, b0, hd**-0.5, softcap=9.0, window=60)


@pytest.mark.parametrize("softcap", [69.0, 70.0, 1000.0])
@pytest.mark.parametrize("heads,kvh,hd,t,base", [(32, 2, 256, 1, [500]), (32, 2, 256, 40, [9]), (16, 4, 128, 12, [3000])])
def test_wide_caps(dev, heads, kvh, hd, t, base, softcap) -> None:
    """Either side of the widest cap whose scores need no running maximum."""
    q, k, v, table, b0 = case(1, 1, t, heads, kvh, hd, base, q_std=8.0)
    check(dev, q, k, v, table, b0, hd**-0.5, softcap=softcap)
    check(dev, q, k, v, table, b0, hd**-0.5, softcap=softcap, slopes=torch.linspace(0.0, 2.0, heads))


@pytest.mark.parametrize("softcap", [1e4, 1e5, 1e8, 1e30, 3e38])
@pytest.mark.parametrize("heads,kvh,hd,t,base", [(32, 2, 256, 1, [500]), (32, 2, 256, 40, [9]), (16, 4, 128, 12, [3000])])
def test_caps_far_above_the_scores(dev, heads, kvh, hd, t, base, softcap) -> None:
    """A cap that is as good as none leaves the scores' own digits. So do the rows that are done again one by one:
    an infinite value that another row sees."""
    for q_std in (2.0, 8.0):
        q, k, v, table, b0 = case(1, 1, t, heads, kvh, hd, base, q_std=q_std)
        check(dev, q, k, v, table, b0, hd**-0.5, softcap=softcap)
    check(dev, q, k, v, table, b0, hd**-0.5, softcap=softcap, slopes=torch.linspace(0.0, 2.0, heads))
    if t > 1:
        at = base[0] + t - 1
        v[int(table[0, at // 16]) * 16 + at % 16] = float("inf")
        want, spread = ref.paged_attention_masked(q[:, :-1], k, v.nan_to_num(0, 0, 0), table, b0, hd**-0.5, softcap=softcap)
        got = run(dev, q, k, v, table, b0, hd**-0.5, softcap=softcap).double().cpu()[:, :-1]
        assert float(((got - want).abs() / bars(want, spread)).max()) <= 1.0


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(8, 2, 64, 1, [40]), (16, 4, 128, 9, [40]), (32, 2, 256, 40, [9])])
def test_caps_far_below_the_scores(dev, heads, kvh, hd, t, base) -> None:
    """All weights equal, those of scores of 0 among them; a cap that float32 does not hold is refused."""
    q, k, v, table, b0 = case(1, 1, t, heads, kvh, hd, base)
    q[:, :, 1] = 0
    k[::3] = 0
    for softcap in (1e-6, 1e-13, 1e-20, 1e-30, 1e-38, 1e-42):
        check(dev, q, k, v, table, b0, hd**-0.5, softcap=softcap)
    with pytest.raises(ValueError):
        run(dev, q, k, v, table, b0, hd**-0.5, softcap=1e-50)


def test_scores_of_a_wide_caps_size(dev) -> None:
    """Scores around and above a quarter of caps of some hundreds, where the cap's two forms meet."""
    for softcap in (100.0, 400.0):
        q, k, v, table, b0 = case(1, 1, 9, 16, 4, 128, [90], q_std=softcap / 8)
        check(dev, q, k, v, table, b0, 128**-0.5, softcap=softcap)


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(32, 2, 256, 1, [500]), (32, 2, 256, 40, [9]), (16, 4, 128, 12, [3000])])
@pytest.mark.parametrize("softcap", [0.0, 30.0, 50.0, 69.0])
def test_scores_far_from_zero(dev, heads, kvh, hd, t, base, softcap) -> None:
    """All scores at the cap's lower or upper end (without a cap: at -3e4 and 3e4): weights are what differences
    between them make, however small or large all of them are."""
    q, k, v, table, b0 = case(2, 1, t, heads, kvh, hd, base)
    far = torch.randn(1, kvh, hd).bfloat16()
    k = (far + torch.randn(k.shape) * 0.02).bfloat16()
    for sign in (1.0, -1.0):
        qs = (sign * far.float().repeat_interleave(heads // kvh, 1) * 16.0).bfloat16().expand(1, t, heads, hd).contiguous()
        check(dev, qs, k, v, table, b0, 1.0 if softcap else hd**-0.5, softcap=softcap)


def test_biases_that_leave_little(dev) -> None:
    """Rows that see only keys far ahead of them (a prefix, their document beginning behind them), so that the
    bias takes every weight far down, and slopes below zero, which take them up."""
    heads, kvh, hd, t = 8, 2, 128, 200
    q, k, v, table, b0 = case(3, 1, t, heads, kvh, hd, [0])
    pos = torch.arange(t)[None]
    first = torch.where(pos < 100, pos + 90, pos - 3)
    slopes = torch.tensor([0.0, 0.1, 0.6, 0.8, 0.9, 1.0, 2.0, 50.0])
    for softcap in (0.0, 50.0):
        check(dev, q, k, v, table, b0, hd**-0.5, softcap=softcap, slopes=slopes, first=first, prefix=b0 + t)
        check(dev, q, k, v, table, b0, hd**-0.5, softcap=softcap, slopes=-slopes[:1].expand(8) - 1.5)


@pytest.mark.parametrize("t,base", [(1, [3000]), (1, [200]), (12, [1500]), (40, [700])])
def test_biases_that_pass_the_range_of_the_sum(dev, t, base) -> None:
    """Slopes below zero whose largest weight is about 2^127, so that every weight and product is finite but their
    sum is not: values are small."""
    heads, kvh, hd = 8, 2, 128
    q, k, v, table, b0 = case(4, 1, t, heads, kvh, hd, base, q_std=0.05)
    slopes = -torch.linspace(120.0, 130.0, heads) * math.log(2.0) / base[0]
    check(dev, q, k, (v.float() * 2.0**-30).bfloat16(), table, b0, hd**-0.5, softcap=50.0, slopes=slopes)


@pytest.mark.parametrize("t,base,heads,kvh,hd", [(1, [29999, 7], 8, 2, 128), (4, [8000, 0, 515], 32, 2, 256), (20, [9000], 8, 2, 64)])
def test_many_key_splits(dev, t, base, heads, kvh, hd) -> None:
    q, k, v, table, b0 = case(9, len(base), t, heads, kvh, hd, base)
    check(dev, q, k, v, table, b0, 0.09, softcap=50.0)
    gate = torch.randn(len(base), t, heads, hd).bfloat16()
    check(dev, q, k, v, table, b0, 0.09, window=2500, gate=gate)
    first = torch.tensor(base)[:, None] + torch.arange(t) - 3  # a document of a few keys, its splits but one empty
    check(dev, q, k, v, table, b0, 0.09, first=first.clamp_min(0))


def test_a_bound_above_and_below_the_context(dev) -> None:
    """The context bound sizes the splits alone."""
    q, k, v, table, b0 = case(4, 2, 3, 8, 2, 128, [900, 40], spare=200)
    want, spread = ref.paged_attention_masked(q, k, v, table, b0, 0.1)
    for ctx in (0, 1, 903, table.shape[1] * 16):
        got = run(dev, q, k, v, table, b0, 0.1, ctx).double().cpu()
        assert torch.all((got - want).abs() <= bars(want, spread))


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(32, 2, 256, 1, [40]), (16, 4, 128, 9, [40]), (32, 2, 256, 40, [40]), (8, 2, 64, 3, [4000])])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), 3.3e38])
def test_unseen_keys_may_hold_anything(dev, heads, kvh, hd, t, base, value) -> None:
    """Rows of the cache that a row does not see never reach it: behind the window, before the document, past
    the last row, later rows of the same call."""
    q, k, v, table, b0 = case(6, 1, t, heads, kvh, hd, base)
    first = torch.full((1, t), base[0] - 9)
    clean = check(dev, q, k, v, table, b0, hd**-0.5, first=first)
    at = torch.arange(table.shape[1] * 16)
    rows = table[0].long()[at // 16] * 16 + at % 16
    unseen = rows[(at < base[0] - 9) | (at >= base[0] + t)]
    k[unseen], v[unseen] = value, value
    k[:16], v[:16] = value, value
    assert torch.equal(run(dev, q, k, v, table, b0, hd**-0.5, first=first).double().cpu(), clean)
    if t > 1:  # the last row's own key and value: the earlier rows are done without them, as the oracle does them
        want, spread = ref.paged_attention_masked(q[:, :-1], k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0), table, b0, hd**-0.5,
                                                  first=first[:, :-1])
        k[rows[base[0] + t - 1]], v[rows[base[0] + t - 1]] = value, value
        got = run(dev, q, k, v, table, b0, hd**-0.5, first=first).double().cpu()[:, :-1]
        worst = float(((got - want).abs() / bars(want, spread)).max())
        assert worst <= 1.0  # and no NaN


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(32, 2, 256, 1, [40]), (16, 4, 128, 9, [40]), (32, 2, 256, 40, [40]), (8, 2, 64, 3, [4000]),
                                                 (16, 4, 128, 60, [90])])
@pytest.mark.parametrize("softcap,slope", [(30.0, 0.0), (50.0, 0.01), (300.0, 0.0), (1e6, 0.0)])
def test_unseen_keys_leave_capped_rows_bit_for_bit(dev, heads, kvh, hd, t, base, softcap, slope) -> None:
    """Finite keys that no row sees, before the document and behind the last row, whose scores lie in the middle of the
    cap's range or at its end: the form in which a tile's scores are capped does not go by them."""
    q, k, v, table, b0 = case(6, 1, t, heads, kvh, hd, base)
    first = torch.full((1, t), base[0] - 9)
    kw = dict(first=first, softcap=softcap, **({"slopes": torch.full((heads,), slope)} if slope else {}))
    clean = check(dev, q, k, v, table, b0, hd**-0.5, **kw)
    at = torch.arange(table.shape[1] * 16)
    unseen = table[0].long()[at // 16] * 16 + at % 16
    unseen = unseen[(at < base[0] - 9) | (at >= base[0] + t)]
    for value in (0.0, 3.0, 8.0, 30.0, 1e4, 1e30):
        k2, v2 = k.clone(), v.clone()
        k2[unseen], v2[unseen] = (k[unseen].float() * value).bfloat16(), 7.0
        assert torch.equal(run(dev, q, k2, v2, table, b0, hd**-0.5, **kw).double().cpu(), clean)


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(8, 2, 64, 3, [40]), (32, 2, 256, 6, [100]), (16, 4, 128, 60, [7]), (8, 2, 128, 1, [5000])])
def test_seen_infinities_and_nan(dev, heads, kvh, hd, t, base) -> None:
    """What a row sees reaches it: an infinite value its channel alone, a NaN key every channel; the rows
    that do not see them stay as they are."""
    q, k, v, table, b0 = case(7, 1, t, heads, kvh, hd, base)
    at = base[0] + t // 2
    row = int(table[0, at // 16]) * 16 + at % 16
    v[row, 0, 5], v[row, 0, 6], v[row, 1, 7] = float("inf"), float("-inf"), float("nan")
    got = run(dev, q, k, v, table, b0, hd**-0.5).double().cpu()
    want, spread = ref.paged_attention_masked(q, k, v, table, b0, hd**-0.5)
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf())
    assert torch.equal(got.isneginf(), want.isneginf()) and bool((~fine).any())
    assert torch.all((got - want).abs()[fine] <= bars(want, spread)[fine])
    v[row] = 1.0
    k[row, 0, 3] = float("nan")
    got = run(dev, q, k, v, table, b0, hd**-0.5, softcap=30.0).double().cpu()
    group = heads // kvh
    assert got[0, t // 2 :, :group].isnan().all() and got[0, : t // 2].isfinite().all() and got[0, :, group:].isfinite().all()


def test_keys_at_minus_infinity(dev) -> None:
    """A seen key at -inf weighs nothing beside others and makes a row of its own NaN, as its softmax is; a
    row that sees no key is zeros."""
    q, k, v, table, b0 = case(8, 1, 3, 8, 2, 64, [20])
    q = q.abs()
    row = [int(table[0, j // 16]) * 16 + j % 16 for j in range(23)]
    k[row[21]] = float("-inf")
    first = torch.tensor([[21, 21, 5]])
    got = run(dev, q, k, v, table, b0, 0.1, first=first).double().cpu()
    assert not got[0, 0].any() and got[0, 1].isnan().all()
    k2 = k.clone()
    k2[row[21]] = -3e38
    want, spread = ref.paged_attention_masked(q, k2, v, table, b0, 0.1, first=first)
    assert torch.all((got - want).abs()[0, 2] <= bars(want, spread)[0, 2])


def test_lanes_that_hold_nothing(dev) -> None:
    """Padding lanes: a negative base, a base past the table, a table entry outside the pool."""
    q, k, v, table, b0 = case(10, 4, 2, 8, 2, 64, [50, 50, 50, 50])
    b0[1], b0[2] = -2, table.shape[1] * 16 + 100
    table[3, 1], table[3, 2] = -5, 2**31 - 1
    got = run(dev, q, k, v, table, b0, 0.1, 52, window=30).double().cpu()
    assert not got[1].any() and not got[2].any()
    k[:16], v[:16] = 0, 0
    table[3, 1] = table[3, 2] = 0  # such blocks read as zeros
    want, spread = ref.paged_attention_masked(q[[0, 3]], k, v, table[[0, 3]], b0[[0, 3]], 0.1, window=30)
    assert torch.all((got[[0, 3]] - want).abs() <= bars(want, spread))


@pytest.mark.parametrize("heads,kvh,hd,t", [(8, 2, 64, 2), (16, 4, 128, 20), (32, 2, 256, 5)])
@pytest.mark.parametrize("past", [1, 2**20, 2**30, 2**31 + 5, 2**40])
def test_a_bias_of_rows_past_the_table(dev, heads, kvh, hd, t, past) -> None:
    """Rows of positions far behind the table's last key: their keys' distances differ as those of near rows do."""
    q, k, v, table, b0 = case(14, 2, t, heads, kvh, hd, [60, 60])
    b0[1] = table.shape[1] * 16 + past
    slopes = torch.linspace(0.01, 0.3, heads)
    q, k, v = q.to(dev), k.to(dev), attention.v_blocks(v).to(dev)
    for kw in ({}, {"softcap": 30.0}):
        got = attention.paged_attention_masked(q, k, v, table.to(dev), b0.to(dev), 80, hd**-0.5, slopes=slopes.to(dev), **kw)
        want, spread = ref.paged_attention_masked(q.cpu(), k.cpu(), attention.v_rows(v).cpu(), table, b0, hd**-0.5, slopes=slopes, **kw)
        assert float(((got.double().cpu() - want).abs() / bars(want, spread)).max()) <= 1.0


def test_strides_and_index_types(dev) -> None:
    q, k, v, table, b0 = case(11, 2, 6, 16, 4, 128, [30, 200])
    kw = dict(prefix=b0 + 3, first=torch.randint(0, 30, (2, 6)))
    want = run(dev, q, k, v, table, b0, 0.1, **kw, gate=q)
    wide = torch.zeros(2, 6, 16, 264).bfloat16().to(dev)
    for at in (0, 8, 1):  # in place, in place, and rows off 16 bytes
        wide[..., at : at + 128] = q.to(dev)
        qq = wide[..., at : at + 128]
        got = run(dev, qq, k, v, table.long(), b0.int(), 0.1, prefix=kw["prefix"].int(), first=kw["first"].int(), gate=qq)
        assert torch.equal(got, want)
    heads_first = q.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
    first = kw["first"].t().contiguous().to(dev).t()
    assert torch.equal(run(dev, heads_first, k, v, table, b0, 0.1, prefix=kw["prefix"], first=first, gate=heads_first), want)


def test_pools_past_four_gigabytes(dev) -> None:
    """Blocks whose byte offsets pass 2^31 and 2^32 in pools whose other rows are never touched."""
    kvh, hd, t = 2, 256, 3
    rows = (2**32 // (kvh * hd * 2) + 4096) // 16 * 16
    q, k, v, table, b0 = case(12, 1, t, 32, kvh, hd, [90])
    kd = torch.empty(rows, kvh, hd, dtype=torch.bfloat16, device=dev)
    vd = torch.empty(rows // 16, kvh, hd, 16, dtype=torch.bfloat16, device=dev)
    far = torch.tensor([[rows // 16 - 1, 2**31 // (kvh * hd * 32), 5, 2**32 // (kvh * hd * 32), rows // 16 - 2, 9, 10]]).int()
    vb = attention.v_blocks(v).to(dev)
    for i in range(table.shape[1]):
        a, b = int(table[0, i]), int(far[0, i])
        kd[b * 16 : b * 16 + 16] = k[a * 16 : a * 16 + 16].to(dev)
        vd[b] = vb[a]
    want = run(dev, q, k, v, table, b0, 0.07, window=80)
    for tt in (1, t):
        got = attention.paged_attention_masked(q[:, -tt:].to(dev), kd, vd, far[:, : table.shape[1]].to(dev),
                                               (b0 + t - tt).to(dev), 93, 0.07, window=80)
        off = (got.double() - want[:, -tt:].double()).abs().cpu()
        assert torch.all(off <= 2.0**-7 * want[:, -tt:].double().cpu().abs() + 2.0**-9)


@pytest.mark.parametrize("heads,kvh,hd,t,base", [(32, 2, 256, 1, [600, 5000]), (32, 2, 256, 4, [3000, 20]), (16, 4, 128, 70, [100, 0])])
def test_graphs_and_streams(dev, heads, kvh, hd, t, base) -> None:
    """Two captured calls with workspaces of their own, replayed in turn with eager work between."""
    calls = []
    for i in range(2):
        q, k, v, table, b0 = case(20 + i, 2, t, heads, kvh, hd, base)
        args = [x.to(dev) for x in (q, k, attention.v_blocks(v), table, b0)]
        kw = {"softcap": 30.0, "window": 0 if i else 900}
        calls.append((args, kw))
    ctx = max(base) + t + 3
    graphs, outs = [], []
    for args, kw in calls:
        attention.paged_attention_masked(*args, ctx, 0.08, **kw)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attention.paged_attention_masked(*args, ctx, 0.08, **kw))
        graphs.append(g)
    for step in range(4):
        for args, _ in calls:
            args[0].copy_(torch.randn_like(args[0]))
            if step:
                args[4].add_(1)
        for g in graphs if step % 2 else reversed(graphs):
            g.replay()
        for (args, kw), out in zip(calls, outs):
            assert torch.equal(out, attention.paged_attention_masked(*args, ctx, 0.08, **kw))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = [attention.paged_attention_masked(*args, ctx, 0.08, **kw) for args, kw in calls]
    b = [attention.paged_attention_masked(*args, ctx, 0.08, **kw) for args, kw in calls]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_after_the_rows_of_the_same_round(dev) -> None:
    """The run of a layer: rotation into the cache, then attention over it, step after step, equal to one
    prompt's call over all rows."""
    import rotary

    b, heads, kvh, hd, n = 2, 16, 4, 128, 21
    g = torch.Generator(dev).manual_seed(3)
    rates, m = rotary.frequencies(hd, 1e6, scaling="yarn", factor=4.0, original=4096, device=dev)
    table = torch.arange(1, 2 * b + 1, device=dev).view(b, 2).int()
    q, k, v = (torch.randn(b, n, h, hd, device=dev, generator=g).bfloat16() for h in (heads, kvh, kvh))
    qn, kn = (torch.randn(hd, device=dev, generator=g).bfloat16() * 0.1 for _ in range(2))
    pools = [(torch.zeros(80, kvh, hd, device=dev).bfloat16(), torch.zeros(5, kvh, hd, 16, device=dev).bfloat16()) for _ in range(2)]
    kw = dict(softcap=20.0, window=13)

    def part(pool, a, z):
        base = torch.full((b,), a, device=dev)
        qr = rotary.rotate_to_cache(q[:, a:z], k[:, a:z], v[:, a:z], rates, *pool, table, base, magnitude=m, q_norm=qn, k_norm=kn)
        return attention.paged_attention_masked(qr, *pool, table, base, z, hd**-0.5, **kw)

    whole = part(pools[0], 0, n)
    steps = torch.cat([part(pools[1], a, z) for a, z in ((0, 1), (1, 2), (2, 6), (6, 17), (17, 21))], 1)
    assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1])
    pos = torch.arange(n).expand(b, n)
    qr = rotary.rotate(q, pos.contiguous().to(dev), rates, magnitude=m, w=qn)
    want, spread = ref.paged_attention_masked(qr.cpu(), pools[0][0].cpu(), attention.v_rows(pools[0][1]).cpu(), table.cpu(),
                                              torch.zeros(b, dtype=torch.long), hd**-0.5, **kw)
    for got in (whole, steps):
        assert torch.all((got.double().cpu() - want).abs() <= bars(want, spread))


def test_refusals(dev) -> None:
    q, k, v, table, b0 = case(13, 2, 3, 8, 2, 64, [30, 20])
    a = dict(q=q, k=k, v=v, table=table, base=b0, scale=0.1)

    def call(**kw):
        m = {**a, **{n: x for n, x in kw.items() if n in a}}
        return run(dev, *m.values(), **{n: x for n, x in kw.items() if n not in a})

    call()
    for kw in ({"q": q.float()}, {"q": q[0]}, {"q": q[..., :32]}, {"k": k[:-8], "v": v[:-16]}, {"k": k[:, :1]}, {"k": k.float()},
               {"table": table[:1]}, {"table": table.float()}, {"base": b0[:1]}, {"base": b0.float()}, {"scale": 0.0},
               {"scale": float("inf")}, {"scale": float("nan")}, {"softcap": -1.0}, {"softcap": float("inf")}, {"window": -1},
               {"ctx": 10**6}, {"ctx": -1}, {"gate": q[:, :2]}, {"gate": q.float()}, {"slopes": torch.zeros(7)},
               {"slopes": torch.zeros(8).double()}, {"prefix": torch.zeros(3).long()}, {"prefix": torch.zeros(2)},
               {"first": torch.zeros(2, 2).long()}, {"first": torch.zeros(2, 3)}):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError):
        attention.paged_attention_masked(q, k, attention.v_blocks(v), table, b0, 33, 0.1)
    assert run(dev, q[:0], k, v, table[:0], b0[:0], 0.1, 33).shape == (0, 3, 8, 64)
    with pytest.raises(ValueError):  # heads that the kv heads do not divide
        run(dev, q[:, :, :7], k, v, table, b0, 0.1)
