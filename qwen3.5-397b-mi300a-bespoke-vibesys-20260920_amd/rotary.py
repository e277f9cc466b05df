"""Position rotation of attention heads on the device (`mtpk_rotate`, `mtpk_rotate_to_cache`).

A head's first `2 * len(rates)` channels are pairs, `(i, i + half)` or, interleaved, `(2 i, 2 i + 1)`;
pair i at position p is turned by `p * rates[i]` radians and multiplied by `magnitude`. The angle is
reduced in 64 bits in the kernel, so there is no table of positions to hold and far positions are as
exact as near ones (`rownorm.rmsnorm`'s `rope` takes fp32 tables instead). `frequencies` gives the rates
of a plain, a stretched or a scaled context.

`rotate` turns (and, with a weight, first norms) the heads of one tensor; `rotate_to_cache` the q and k
heads of a round's rows, with k and v into the paged caches, in one launch: what `rownorm.rmsnorm` of q
and of k and `attention.kv_write` do in three. fp32 arithmetic with one rounding at the end. Device
tensors only.
"""

from __future__ import annotations

import math

import torch

import _mtpk


def frequencies(dim: int, theta: float, *, scaling: str = "none", factor: float = 1.0, original: int = 0,
                fast: float = 32.0, slow: float = 1.0,
                device: torch.device | str = "cpu") -> tuple[torch.Tensor, float]:
    """`(rates, magnitude)` of a rotation over `dim` channels: fp64 `[dim / 2]` radians per position on
    `device`, and the factor on the rotated channels.

    `scaling`: "none", `theta ** (-2 i / dim)`; "linear", those over `factor` (positions interpolated);
    "ntk", the same of the base `theta * factor ** (dim / (dim - 2))`, which leaves the fastest pair as it
    is and slows the slowest by `factor`; "yarn", those over `factor` for pairs that turn less than
    `slow` times over the `original` context, unchanged for pairs that turn more than `fast` times, a
    linear ramp over the pair's index between the two, and magnitude `0.1 ln(factor) + 1`."""
    if dim < 2 or dim % 2:
        raise ValueError(f"a rotation takes an even number of channels, got {dim}")
    if not theta > 0 or not factor >= 1:
        raise ValueError(f"theta must be positive and factor at least 1, got {theta} and {factor}")
    half = dim // 2
    index = torch.arange(half, dtype=torch.float64)
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("one pair has no slowest to scale: dim must be over 2")
        theta = theta * factor ** (dim / (dim - 2))
    rates = float(theta) ** (-index / half)
    if scaling in ("none", "ntk"):
        return rates.to(device), 1.0
    if scaling == "linear":
        return (rates / factor).to(device), 1.0
    if scaling != "yarn":
        raise ValueError(f"unknown scaling {scaling!r}")
    if original < 1 or not fast > slow > 0 or theta == 1:
        raise ValueError("yarn takes the original context's length, fast > slow > 0 and a theta other than 1")
    low, high = (half * math.log(original / (2 * math.pi * turns)) / math.log(theta) for turns in (fast, slow))
    low, high = max(math.floor(low), 0), min(math.ceil(high), dim - 1)
    ramp = ((index - low) / max(high - low, 0.001)).clamp(0, 1)
    return (rates / factor * ramp + rates * (1 - ramp)).to(device), 0.1 * math.log(factor) + 1.0


def rotate(x: torch.Tensor, positions: torch.Tensor, rates: torch.Tensor, *, magnitude: float = 1.0,
           interleaved: bool = False, w: torch.Tensor | None = None, eps: float = 1e-6,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Heads `x` `[..., heads, dim]` (fp32 or bf16), normed by `x * rsqrt(mean(x^2) + eps) * (1 + w)` when
    `w` `[dim]` is given, rotated at `positions` (integers of shape `x.shape[:-2]`). Returns a new tensor of
    x's shape and type, or `out` (which may be `x`, but overlap it in no other way). Any strides of x;
    rows that do not lie on 16 bytes are copied first. `dim` is a multiple of 8 up to 512."""
    return _mtpk.native().rotate(x, positions, rates, magnitude, interleaved, w, eps, out, _mtpk.stream_for(x))


def rotate_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rates: torch.Tensor, k_pool: torch.Tensor,
                    v_pool: torch.Tensor, block_table: torch.Tensor, base_pos: torch.Tensor, *,
                    magnitude: float = 1.0, interleaved: bool = False, q_norm: torch.Tensor | None = None,
                    k_norm: torch.Tensor | None = None, eps: float = 1e-6, keep: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None) -> torch.Tensor:
    """A round's rows on their way to attention: q `[B, t, heads, hd]` and k `[B, t, kv_heads, hd]` normed
    (where `q_norm`, `k_norm` are given) and rotated at `base_pos[b] + s`, or at `positions` `[B, t]`; k and v
    stored at `base_pos[b] + s` through `block_table` as `attention.kv_write` stores them, but for rows with
    `keep[b, s]` False. Returns q, contiguous `[B, t, heads, hd]`. bf16; any strides (rows that do not lie on
    16 bytes are copied first). Rows of a lane must not share a pool row with another lane's."""
    return _mtpk.native().rotate_to_cache(q, k, v, rates, k_pool, v_pool, block_table, base_pos, magnitude, interleaved,
                                          q_norm, k_norm, eps, keep, positions, _mtpk.stream_for(q))
