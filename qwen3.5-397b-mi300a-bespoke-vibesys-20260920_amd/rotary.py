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

import ctypes
import math

import torch

import _mtpk
import attention

MAX_DIM = 512


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


_Two, _Three = ctypes.c_int64 * 2, ctypes.c_int64 * 3


def _check_rates(rates: torch.Tensor, dim: int) -> int:
    if rates.dtype != torch.float64 or rates.dim() != 1 or not rates.is_contiguous():
        raise ValueError("rates must be a contiguous float64 [pairs] tensor")
    rot = 2 * rates.shape[0]
    if not 2 <= rot <= dim:
        raise ValueError(f"{rates.shape[0]} pairs do not fit heads of {dim} channels")
    if dim % 8 or dim > MAX_DIM:
        raise ValueError(f"head dim must be a multiple of 8 up to {MAX_DIM}, got {dim}")
    return rot


def _check_norm(w: torch.Tensor, dim: int, device: torch.device) -> tuple[torch.Tensor, int]:
    if w.shape != (dim,) or w.device != device:
        raise ValueError(f"a norm's weight must be a [{dim}] tensor on {device}")
    return w if _mtpk.rows16(w) else w.clone(memory_format=torch.contiguous_format), _mtpk.float_code(w.dtype)


def rotate(x: torch.Tensor, positions: torch.Tensor, rates: torch.Tensor, *, magnitude: float = 1.0,
           interleaved: bool = False, w: torch.Tensor | None = None, eps: float = 1e-6,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Heads `x` `[..., heads, dim]` (fp32 or bf16), normed by `x * rsqrt(mean(x^2) + eps) * (1 + w)` when
    `w` `[dim]` is given, rotated at `positions` (integers of shape `x.shape[:-2]`). Returns a new tensor of
    x's shape and type, or `out` (which may be `x`, but overlap it in no other way). Any strides of x;
    rows that do not lie on 16 bytes are copied first."""
    device = _mtpk.require_device(x, positions, rates)
    if x.dim() < 2 or positions.shape != x.shape[:-2]:
        raise ValueError(f"positions must be {list(x.shape[:-2])} for heads {list(x.shape)}, got {list(positions.shape)}")
    heads, dim = x.shape[-2:]
    rot = _check_rates(rates, dim)
    dtype = _mtpk.float_code(x.dtype)
    w_dtype = 0
    if w is not None:
        w, w_dtype = _check_norm(w, dim, device)
    if positions.dtype != torch.int64:
        if positions.dtype.is_floating_point or positions.dtype.is_complex or positions.dtype == torch.bool:
            raise ValueError("positions must be integers")
        positions = positions.to(torch.int64)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != device:
        raise ValueError(f"out must be {list(x.shape)} {x.dtype} on {device}")
    src, dst = _tokens(x), _tokens(out)
    if src is None:
        src = x.clone(memory_format=torch.contiguous_format).view(-1, heads, dim)
    if dst is None:
        raise ValueError("out's rows must lie on 16 bytes and its leading dims at one stride")
    tokens = src.shape[0]
    if tokens == 0 or heads == 0:
        return out
    pos = positions if positions.is_contiguous() else positions.contiguous()
    xs, os_ = _Two(*src.stride()[:2]), _Two(*dst.stride()[:2])
    with _mtpk.on(device):
        status = _mtpk.lib().mtpk_rotate(
            src.data_ptr(), dtype, ctypes.addressof(xs), tokens, heads, dim, None if w is None else w.data_ptr(),
            w_dtype, eps, pos.data_ptr(), rates.data_ptr(), rot, interleaved, magnitude, dst.data_ptr(),
            ctypes.addressof(os_), _mtpk.stream_of(device))
    if status:
        _mtpk.check(status, "mtpk_rotate")
    return out


def _tokens(x: torch.Tensor) -> torch.Tensor | None:
    """`[..., heads, dim]` as a `[tokens, heads, dim]` view, or None where the leading dims have no one
    stride or the rows do not lie on 16 bytes."""
    if x.dim() != 3:
        heads, dim = x.shape[-2:]
        try:
            x = x.view(-1, heads, dim) if x.numel() else x.reshape(0, heads, dim)
        except RuntimeError:
            return None
    return x if _mtpk.rows16(x) else None


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
    device = _mtpk.require_device(q, k, v, rates, k_pool, v_pool, block_table, base_pos)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"q and k must be [B, t, heads, hd], got {list(q.shape)} and {list(k.shape)}")
    b, t, heads, hd = q.shape
    kvh = k.shape[2]
    if k.shape != (b, t, kvh, hd) or v.shape != k.shape:
        raise ValueError(f"k and v must be [{b}, {t}, kv_heads, {hd}], got {list(k.shape)} and {list(v.shape)}")
    if not q.dtype == k.dtype == v.dtype == torch.bfloat16:
        raise ValueError("q, k and v must be bf16")
    rot = _check_rates(rates, hd)
    table, pos = attention.cache_operands(k_pool, v_pool, block_table, base_pos, b, kvh, hd)
    norm_dtype = 0
    if q_norm is not None:
        q_norm, norm_dtype = _check_norm(q_norm, hd, device)
    if k_norm is not None:
        k_norm, k_dtype = _check_norm(k_norm, hd, device)
        if q_norm is not None and k_dtype != norm_dtype:
            raise ValueError("q_norm and k_norm must be of one type")
        norm_dtype = k_dtype
    if positions is not None:
        if positions.shape != (b, t) or positions.dtype != torch.int64 or positions.device != device:
            raise ValueError(f"positions must be int64 [{b}, {t}] on {device}")
        positions = positions.contiguous()
    kb = ks = 0
    if keep is not None:
        if keep.shape != (b, t) or keep.element_size() != 1 or keep.device != device:
            raise ValueError(f"keep must be bool [{b}, {t}] on {device}")
        kb, ks = keep.stride()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.numel() == 0:
        return out
    q, k, v = (x if _mtpk.rows16(x) else x.clone(memory_format=torch.contiguous_format) for x in (q, k, v))
    st = []
    for x in (q, k, v, out):
        s = x.stride()
        st.append(_Three(s[0], s[2], s[1]))
    qs, ks_, vs, os_ = st
    with _mtpk.on(device):
        status = _mtpk.lib().mtpk_rotate_to_cache(
            q.data_ptr(), ctypes.addressof(qs), k.data_ptr(), ctypes.addressof(ks_), v.data_ptr(), ctypes.addressof(vs),
            _mtpk.ptr(q_norm), _mtpk.ptr(k_norm), norm_dtype, eps, rates.data_ptr(), rot, interleaved, magnitude,
            k_pool.data_ptr(), v_pool.data_ptr(), k_pool.shape[0], table.data_ptr(), table.shape[1], pos.data_ptr(),
            _mtpk.ptr(positions), _mtpk.ptr(keep), kb, ks, b, t, heads, kvh, hd, out.data_ptr(), ctypes.addressof(os_),
            _mtpk.stream_of(device))
    if status:
        _mtpk.check(status, "mtpk_rotate_to_cache")
    return out
