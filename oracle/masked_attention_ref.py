"""Paged attention with capped and biased scores and masks beyond the causal order, in float64 torch on
the CPU. TEST INFRASTRUCTURE ONLY (see oracle/__init__).

For the query row at position p = base[b] + s of q head h and the key at position j of lane b:
  x = scale * q . k_j;  x = softcap * tanh(x / softcap) when softcap > 0;  x -= slopes[h] * |p - j|
  seen iff first[b, s] <= j < base[b] + t, p - j < window (0: none), and j <= p or both below prefix[b]
out = sum over the seen j of softmax(x)_j v_j; zeros where none is seen; times sigmoid(gate).

Pinning (tests/test_oracle_masked_attention.py): without caps, biases and masks it is
`attention_ref.paged_attention`; identical keys give the mean of the values that each mask admits; a cap
far above the scores changes nothing and one far below makes all weights equal; a steep slope leaves the
row's own key.
"""

from __future__ import annotations

import torch


def paged_attention_masked(q, k_pool, v_pool, table, base, scale, *, softcap=0.0, window=0, slopes=None, prefix=None,
                           first=None, gate=None, block: int = 16):
    """q [B, t, heads, hd]; pools [rows, kv_heads, hd]; table [B, blocks]; base [B]. Returns float64 (out,
    spread), both [B, t, heads, hd]: spread is sum_j w_j |v_j| with the row's weights, gated as out is."""
    q, kp, vp = (x.double() for x in (q, k_pool, v_pool))
    b, t, heads, hd = q.shape
    group = heads // kp.shape[1]
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(b):
        end = min(int(base[i]) + t, table.shape[1] * block)
        j = torch.arange(max(end, 0))
        rows = table[i].long()[j // block] * block + j % block
        p = int(base[i]) + torch.arange(t)[:, None]
        seen = j <= p
        if prefix is not None:
            seen = seen | ((p < int(prefix[i])) & (j < int(prefix[i])))
        if window:
            seen = seen & (p - j < window)
        if first is not None:
            seen = seen & (j >= first[i].long()[:, None])
        for h in range(heads):
            x = q[i, :, h] @ kp[rows, h // group].t() * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * (p - j).abs().double()
            x = x.masked_fill(~seen, -torch.inf)
            any_ = seen.any(-1)
            w = torch.softmax(x[any_], -1)
            v = vp[rows, h // group]
            # a key outside the row's set has no part in it, whatever its value is
            odd = ~torch.isfinite(v)
            o = w @ v.masked_fill(odd, 0.0)
            if bool(odd.any()):
                s = seen[any_].double()
                up, down = (((v == sign * torch.inf) | v.isnan()).double() for sign in (1, -1))
                o = o + torch.where(s @ up > 0, torch.inf, 0.0) - torch.where(s @ down > 0, torch.inf, 0.0)
            out[i, any_, h] = o
            spread[i, any_, h] = w @ v.masked_fill(odd, 0.0).abs()
    if gate is not None:
        out, spread = (x * torch.sigmoid(gate.double()) for x in (out, spread))
    return out, spread
