"""The operators of a verified tree of drafts, in float64 on the CPU. TEST INFRASTRUCTURE ONLY (see oracle/__init__).

A tree is one lane's `parents` [t]: node s hangs below the earlier node parents[s], or below the committed context at -1;
any other value, and what hangs below such a node, is absent. Every operator is stated along a node's way, the node with
its ancestors from the root down, as the chain's own oracle runs it: `deltanet_ref.delta_rule_step` for the rule, a causal
convolution for its inputs, attention over the context and the way's keys.

Pinning (tests/test_oracle_tree.py): on a chain every operator is the chain's oracle; a node's result does not change when
nodes off its way do; acceptance of a chain is `accept_ref`'s; a path that is already in place moves nothing.
"""

from __future__ import annotations

import numpy as np
import torch

from oracle import deltanet_ref


def ways(parents) -> list[list[int] | None]:
    """Each node's way from the root, None where it is absent."""
    out: list[list[int] | None] = []
    for s, p in enumerate(int(p) for p in parents):
        if p < -1 or p >= s or (p >= 0 and out[p] is None):
            out.append(None)
        else:
            out.append((out[p] if p >= 0 else []) + [s])
    return out


def attention(q, k_pool, v_pool, table, base, scale, parents, gate=None, block: int = 16):
    """q [B, t, heads, hd]; pools [rows, kv_heads, hd]; table [B, blocks]; base [B]; parents [B, t]. Returns float64 (out,
    spread), both [B, t, heads, hd]: spread is sum_j w_j |v_j| with the row's weights, gated as out is. Positions past
    the table are not seen."""
    q, kp, vp = (x.double() for x in (q, k_pool, v_pool))
    b, t, heads, hd = q.shape
    group = heads // kp.shape[1]
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(b):
        end = table.shape[1] * block
        for s, way in enumerate(ways(parents[i])):
            if way is None:
                continue
            j = torch.tensor([x for x in [*range(int(base[i])), *(int(base[i]) + a for a in way)] if x < end], dtype=torch.long)
            if not len(j):
                continue
            rows = table[i].long()[j // block] * block + j % block
            for h in range(heads):
                w = torch.softmax(kp[rows, h // group] @ q[i, s, h] * scale, -1)
                out[i, s, h] = w @ vp[rows, h // group]
                spread[i, s, h] = w @ vp[rows, h // group].abs()
    if gate is not None:
        present = torch.tensor([[w is not None for w in ways(p)] for p in parents])[..., None, None]
        out, spread = (torch.where(present, x * torch.sigmoid(gate.double()), 0.0) for x in (out, spread))
    return out, spread


def delta_rule(state, slots, q, k, v, g, beta, parents) -> np.ndarray:
    """`deltanet_ref.delta_rule_rows`'s operands without lengths; parents [B, t]. Every node's output, zeros where absent
    or where the slot lies outside the pool."""
    b, t, heads, dv = v.shape
    rep = heads // q.shape[2]
    out = np.zeros((b, t, heads, dv))
    for j in range(b):
        if not 0 <= int(slots[j]) < state.shape[0]:
            continue
        for h in range(heads):
            after: dict[int, np.ndarray] = {-1: np.asarray(state[int(slots[j]), h], np.float64)}
            for s, way in enumerate(ways(parents[j])):
                if way is not None:
                    above = way[-2] if len(way) > 1 else -1
                    after[s], out[j, s, h] = deltanet_ref.delta_rule_step(
                        after[above], q[j, s, h // rep], k[j, s, h // rep], v[j, s, h], g[j, s, h], beta[j, s, h])
    return out


def commit(state, conv, slots, k, v, g, beta, path, lengths, raw) -> tuple[np.ndarray, np.ndarray]:
    """The state pool and the conv windows [slots, C, k1] after each row's path; raw [B, t, C]."""
    state, conv = np.array(state, np.float64), np.array(conv, np.float64)
    b, t, heads, _ = v.shape
    rep, k1 = heads // k.shape[2], conv.shape[2]
    for j in range(b):
        slot = int(slots[j])
        if not 0 <= slot < state.shape[0]:
            continue
        way = []
        for i in range(min(max(int(lengths[j]), 0), t)):
            if not 0 <= int(path[j][i]) < t:
                break
            way.append(int(path[j][i]))
        for i in way:
            for h in range(heads):
                state[slot, h], _ = deltanet_ref.delta_rule_step(state[slot, h], k[j, i, h // rep], k[j, i, h // rep],
                                                                 v[j, i, h], g[j, i, h], beta[j, i, h])
        columns = np.concatenate([conv[slot], np.asarray(raw[j], np.float64)[way].T], axis=1)
        conv[slot] = columns[:, -k1:]
    return state, conv


def conv_rows(conv, slots, conv_w, raw, parents) -> np.ndarray:
    """The causal convolution's sums [B, t, C] along each node's way, before the SiLU; zeros where absent, a zero window for
    a slot outside the pool. conv [slots, C, k1], conv_w [C, k1 + 1], raw [B, t, C]."""
    conv, conv_w, raw = (np.asarray(x, np.float64) for x in (conv, conv_w, raw))
    out = np.zeros(raw.shape)
    for j in range(raw.shape[0]):
        inside = 0 <= int(slots[j]) < conv.shape[0]
        stored = conv[int(slots[j])] if inside else np.zeros(conv.shape[1:])
        for s, way in enumerate(ways(parents[j])):
            if way is not None:
                columns = np.concatenate([stored, raw[j][way].T], axis=1)[:, -conv_w.shape[1] :]
                out[j, s] = (columns * conv_w).sum(1)
    return out


def accept(best, tokens, parents, active, pos, budget, stops) -> dict[str, list]:
    """Python lists in, lists out: the names of `graph_mtp.TreeAccept`."""
    names = ("path", "accept_len", "lengths", "keep", "bonus", "next_pos", "budget_left", "live", "hidden_src")
    out: dict[str, list] = {n: [] for n in names}
    for j, row in enumerate(best):
        t, way, present = len(row), [0], ways(parents[j])
        while len(way) < budget[j] and row[way[-1]] not in stops[j]:
            below = [s for s in range(way[-1] + 1, t) if parents[j][s] == way[-1] and present[s] and tokens[j][s] == row[way[-1]]]
            if not below:
                break
            way.append(below[0])
        n, bonus = len(way) - 1, row[way[-1]]
        values = (way + [way[-1]] * (t - len(way)), n, n + 1 if active[j] else 1, [active[j] and i <= n for i in range(t)],
                  bonus, pos[j] + n + 1, budget[j] - n - 1, bonus not in stops[j] and budget[j] > n + 1, j * t + way[-1])
        for name, value in zip(names, values, strict=True):
            out[name].append(value)
    return out


def keep_rows(k_rows, table, base, path, lengths, block: int = 16):
    """Rows `[pool rows, ...]` after the accepted ones have moved (for K, and for V as rows)."""
    new = k_rows.clone()
    for j in range(len(base)):
        at = lambda x: int(table[j][x // block]) * block + x % block  # noqa: E731
        for i in range(int(lengths[j])):
            new[at(int(base[j]) + i)] = k_rows[at(int(base[j]) + int(path[j][i]))]
    return new
