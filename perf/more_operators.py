"""The operators that verify a tree of drafts whose speed is measured: paged attention of a tree's nodes,
the DeltaNet rows' preparation and gated delta rule along each node's own path, the acceptance of one path
with its cache rows, and the recurrent state's advance along it.

`listed()` names the cases; `draw(rng)` gives more of the same ranges; `prepare(case, seed)` makes what
a serving program holds before the call; `run(state)` makes one pass, through the package's entry points
where `own` is true and in elementary torch operations otherwise; `exact(case, seed)` computes the same
outputs in 64 bits from the definitions; `work(case)` counts what a pass cannot do without.

A tree is `parents` `[B, t]`: node 0 is the lane's own token (parent -1), node s hangs below an earlier
one, and -2 marks the nodes past the end of a lane's smaller tree. Node s of lane b keeps its key and value
at cache position `base[b] + s`.
"""

import math
import sys
from pathlib import Path

import torch

PKG = Path.cwd() / "qwen3.5-397b-mi300a-bespoke-vibesys-20260920_amd"

own = False

DEV = "cuda:0"
BLOCK = 16  # rows of a cache block
LAYOUTS = {256: (32, 2), 128: (16, 4), 64: (8, 2)}  # head_dim -> q heads, kv heads
KD = 128  # key and value channels of a DeltaNet head
CONV = 4  # taps of its causal convolution
EPS = 1e-6
VOCAB = 248320


def listed():
    return [
        # One user's small tree over a short chat, smallest heads: all latency.
        {"name": "attn_tree_1", "kind": "attention", "batch": 1, "nodes": 7, "head_dim": 64, "least": 299, "most": 299,
         "gate": False},
        # The attention layer of 48 users, trees of up to 16 drafts, output gated.
        {"name": "attn_tree_48", "kind": "attention", "batch": 48, "nodes": 16, "head_dim": 256, "least": 2000, "most": 4090,
         "gate": True},
        # Two users' large trees over long contexts.
        {"name": "attn_tree_long_2", "kind": "attention", "batch": 2, "nodes": 63, "head_dim": 128, "least": 31000,
         "most": 65001, "gate": False},
        # One user's rows on their way to the delta rule: all latency.
        {"name": "prep_tree_1", "kind": "prep", "batch": 1, "nodes": 7, "k_heads": 16, "v_heads": 64, "dtype": "bf16"},
        # The same of 48 users.
        {"name": "prep_tree_48", "kind": "prep", "batch": 48, "nodes": 16, "k_heads": 16, "v_heads": 64, "dtype": "bf16"},
        # The delta rule of one user's small tree.
        {"name": "rule_tree_1", "kind": "rule", "batch": 1, "nodes": 7, "k_heads": 16, "v_heads": 64},
        # Of 48 users' trees, bound by their states.
        {"name": "rule_tree_48", "kind": "rule", "batch": 48, "nodes": 16, "k_heads": 16, "v_heads": 64},
        # Of a dozen users' large trees.
        {"name": "rule_tree_12", "kind": "rule", "batch": 12, "nodes": 61, "k_heads": 16, "v_heads": 64},
        # One user's state along the accepted path.
        {"name": "commit_path_1", "kind": "commit", "batch": 1, "nodes": 7, "longest": 4, "k_heads": 16, "v_heads": 64,
         "dtype": "bf16"},
        # The same of 48 users, 1 to 6 accepted nodes each.
        {"name": "commit_path_48", "kind": "commit", "batch": 48, "nodes": 16, "longest": 6, "k_heads": 16, "v_heads": 64,
         "dtype": "bf16"},
        # One user's acceptance, and the accepted nodes' rows moved together in the caches of 15 layers.
        {"name": "take_path_1", "kind": "take", "batch": 1, "nodes": 7, "longest": 4, "head_dim": 256, "least": 299,
         "most": 299, "layers": 15},
        # The same of 48 users with large trees.
        {"name": "take_path_48", "kind": "take", "batch": 48, "nodes": 61, "longest": 8, "head_dim": 256, "least": 150,
         "most": 500, "layers": 15},
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "prep", "rule", "rule", "commit", "take"))
    nodes = rng.choice((_log_int(rng, 1, 64), rng.randint(2, 32)))
    if kind == "attention":
        most = _log_int(rng, 1, 40000) - 1
        batch = _log_int(rng, 1, max(1, min(64, 3_000_000 // ((most + 64) * nodes))))
        return {"kind": kind, "batch": batch, "nodes": nodes, "head_dim": rng.choice((256, 256, 128, 64)),
                "least": rng.randint(most // 4, most), "most": most, "gate": rng.random() < 0.5}
    k_heads, v_heads = rng.choice(((16, 64), (16, 64), (16, 32), (8, 16), (4, 4)))
    if kind == "take":
        least = _log_int(rng, 1, 300) - 1
        return {"kind": kind, "batch": _log_int(rng, 1, 48), "nodes": nodes, "longest": rng.randint(1, min(nodes, 9)),
                "head_dim": rng.choice((256, 256, 128, 64)), "least": least, "most": least + rng.randint(0, 200),
                "layers": rng.randint(1, 15)}
    batch = _log_int(rng, 1, max(1, min(48, 770 // nodes)))
    case = {"kind": kind, "batch": batch, "nodes": nodes, "k_heads": k_heads, "v_heads": v_heads}
    if kind == "commit":
        case["longest"] = rng.randint(1, min(nodes, 9))
    if kind != "rule":
        case["dtype"] = rng.choice(("bf16", "bf16", "f32"))
    return case


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def _bases(c):
    """The lanes' cached positions before the call: ragged from `least` to `most`."""
    return [c["most"] - (c["most"] - c["least"]) * (37 * b % 61) // 60 for b in range(c["batch"])]


def _sizes(c):
    """The lanes' tree sizes: from three quarters of `nodes` up."""
    return [c["nodes"] - (5 * b) % (c["nodes"] // 4 + 1) for b in range(c["batch"])]


def _lengths(c):
    """The lanes' accepted nodes, their own token among them."""
    return [min(1 + (c["longest"] - 1 + 5 * b) % c["longest"], n) for b, n in enumerate(_sizes(c))]


def _parents(gen, c):
    b, t = c["batch"], c["nodes"]
    at = torch.arange(t, device=DEV)
    p = (torch.rand(b, t, generator=gen, device=DEV) * at).long()
    p = torch.minimum(p, at - 1)
    return torch.where(at < torch.tensor(_sizes(c), device=DEV)[:, None], p, -2).int()


def _paths(gen, c):
    """Rising node ids from 0, `_lengths` of them a lane and its last one repeated behind."""
    t = c["nodes"]
    sizes, lengths = (torch.tensor(x, device=DEV)[:, None] for x in (_sizes(c), _lengths(c)))
    at = torch.arange(t, device=DEV)
    key = torch.rand(c["batch"], t, generator=gen, device=DEV) + (at >= sizes) * 2.0
    key[:, 0] = -1.0
    path = torch.where(at < lengths, key.argsort(1), t).sort(1).values
    return torch.where(at < lengths, path, path.gather(1, lengths - 1))


def _tables(gen, c):
    """The lanes' block tables over a shuffled pool, block 0 in no lane's hands."""
    per = -(-(c["most"] + c["nodes"]) // BLOCK)
    n = c["batch"] * per + 1
    order = torch.randperm(n - 1, generator=gen, device=DEV) + 1
    return n, order.view(c["batch"], per).int()


def prepare(case, seed):
    c, gen = case, _gen(seed)
    b, t = c["batch"], c["nodes"]
    s = {"case": c, "parents": _parents(gen, c)}
    if c["kind"] in ("attention", "take"):
        heads, kvh = LAYOUTS[c["head_dim"]]
        hd = c["head_dim"]
        n, s["table"] = _tables(gen, c)
        s["base"] = torch.tensor(_bases(c), device=DEV)
    if c["kind"] == "attention":
        s["k_pool"] = _normal(gen, n * BLOCK, kvh, hd)
        s["v_pool"] = _normal(gen, n, kvh, hd, BLOCK)
        s["q"] = _normal(gen, b, t, heads, hd)
        # the gate as the projection leaves it, beside the query of each head
        s["gate"] = _normal(gen, b, t, heads, 2 * hd)[..., hd:] if c["gate"] else None
        return s
    if c["kind"] == "take":
        s["k"] = _normal(gen, c["layers"], n * BLOCK, kvh, hd)
        s["v"] = _normal(gen, c["layers"], n, kvh, hd, BLOCK)
        s["pools"] = [*s["k"].unbind(0), *s["v"].unbind(0)]
        path, lengths = _paths(gen, c), torch.tensor(_lengths(c), device=DEV)
        parents, tokens = s["parents"], torch.randint(0, VOCAB, (b, t), generator=gen, device=DEV)
        best = torch.randint(0, VOCAB, (b, t), generator=gen, device=DEV)
        for i in range(1, t):  # the path's nodes hang below each other, and the model agrees with them
            on, at, above = i < lengths, path[:, i : i + 1], path[:, i - 1 : i]
            parents.scatter_(1, at, torch.where(on[:, None], above.int(), parents.gather(1, at)))
            best.scatter_(1, above, torch.where(on[:, None], tokens.gather(1, at), best.gather(1, above)))
        last = path[:, -1:]
        best.scatter_(1, last, torch.randint(VOCAB, VOCAB + 500, (b, 1), generator=gen, device=DEV))  # a token of no draft
        s.update(tokens=tokens, best=best, active=torch.arange(b, device=DEV) % 11 != 10, pos=s["base"].clone(),
                 budget=torch.where(torch.arange(b, device=DEV) % 7 == 3, 2, 200))
        s["stops"] = torch.full((b, 8), -1, dtype=torch.long, device=DEV)
        s["stops"][:, 0] = VOCAB + 7
        return s
    kh, vh = c["k_heads"], c["v_heads"]
    slots = b + 3
    s["slots"] = torch.randperm(slots, generator=gen, device=DEV)[:b]
    rates = (torch.rand(vh, generator=gen, device=DEV) * 15.0 + 0.02).log()
    if c["kind"] != "rule":  # the projection's row: q, k and v channels, the gate z, beta and the decay
        dt = torch.float32 if c["dtype"] == "f32" else torch.bfloat16
        s["channels"] = 2 * kh * KD + vh * KD
        s["proj"] = _normal(gen, b, t, s["channels"] + vh * KD + 2 * vh, dtype=dt)
        s["conv"] = _normal(gen, slots, s["channels"], CONV - 1, dtype=dt)
    if c["kind"] == "prep":
        s["conv_w"] = _normal(gen, s["channels"], CONV, std=0.3, dtype=dt)
        s["a_log"], s["dt_bias"] = rates, torch.rand(vh, generator=gen, device=DEV)
        return s
    f32 = torch.float32
    q, k = (_normal(gen, b, t, kh, KD, dtype=f32) for _ in range(2))
    s["q"] = q / q.norm(dim=-1, keepdim=True) * KD**-0.5
    s["k"] = k / k.norm(dim=-1, keepdim=True)
    s["v"] = _normal(gen, b, t, vh, KD, dtype=f32)
    s["g"] = -rates.exp() * torch.log1p(_normal(gen, b, t, vh, dtype=f32).sub(1.0).exp())
    s["beta"] = torch.sigmoid(_normal(gen, b, t, vh, dtype=f32))
    s["state"] = _normal(gen, slots, vh, KD, KD, std=0.3, dtype=f32)
    if c["kind"] == "commit":
        s["path"], s["lengths"] = _paths(gen, c), torch.tensor(_lengths(c), device=DEV)
    return s


# ---------------------------------------------------------------- one pass


def run(state):
    kind = state["case"]["kind"]
    return globals()[f"_{'own' if own else 'plain'}_{kind}"](state)


def _package():
    if str(PKG) not in sys.path:
        sys.path.insert(0, str(PKG))
    import attention
    import deltanet
    import graph_mtp

    return attention, deltanet, graph_mtp


def _own_attention(s):
    attention, _, _ = _package()
    c = s["case"]
    return attention.paged_attention_tree(s["q"], s["k_pool"], s["v_pool"], s["table"], s["base"], c["most"] + c["nodes"],
                                          c["head_dim"] ** -0.5, s["parents"], gate=s["gate"])


def _own_prep(s):
    _, deltanet, _ = _package()
    c = s["case"]
    q, k, v, g, beta = deltanet.prep_tree(s["proj"], s["conv"], s["slots"], s["conv_w"], s["a_log"], s["dt_bias"], c["k_heads"],
                                          KD, c["v_heads"], KD, s["parents"], EPS)
    return {"q": q, "k": k, "v": v, "g": g, "beta": beta}


def _own_rule(s):
    _, deltanet, _ = _package()
    return deltanet.delta_rule_tree(s["state"], s["slots"], s["q"], s["k"], s["v"], s["g"], s["beta"], s["parents"])


def _own_commit(s):
    _, deltanet, _ = _package()
    deltanet.commit_path(s["state"], s["conv"], s["slots"], s["k"], s["v"], s["g"], s["beta"], s["path"], s["lengths"],
                         s["proj"], s["channels"])
    return {"state": s["state"], "conv": s["conv"]}


def _own_take(s):
    attention, _, graph_mtp = _package()
    r = graph_mtp.tree_accept(s["best"], s["tokens"], s["parents"], s["active"], s["pos"], s["budget"], s["stops"])
    attention.keep_path(s["pools"], s["table"], s["base"], r.path, r.lengths)
    return {"path": r.path, "accept_len": r.accept_len, "lengths": r.lengths, "keep": r.keep, "bonus": r.bonus,
            "next_pos": r.next_pos, "budget_left": r.budget_left, "live": r.live, "hidden_src": r.hidden_src,
            "k": s["k"], "v": s["v"]}


def _ancestors(parents):
    """`[B, t, t]`: whether node j lies on the way to node i (i itself included); empty rows for absent nodes."""
    t = parents.shape[1]
    rows = []
    for i in range(t):
        p = parents[:, i].long()
        row = torch.zeros(parents.shape[0], t, dtype=torch.bool, device=DEV)
        if i:
            row = torch.stack(rows, 1).gather(1, p.clamp(min=0)[:, None, None].expand(-1, 1, t))[:, 0]
        row = row & (p >= 0)[:, None]
        row[:, i] = p >= -1
        rows.append(row)
    return torch.stack(rows, 1)


def _plain_attention(s):
    c = s["case"]
    b, t, heads, hd = s["q"].shape
    kvh = s["k_pool"].shape[1]
    group, n = heads // kvh, s["table"].shape[1] * BLOCK
    k = s["k_pool"].view(-1, BLOCK, kvh, hd)[s["table"].long()].float().view(b, n, kvh, hd)
    v = s["v_pool"][s["table"].long()].float()  # [b, blocks, kvh, hd, BLOCK]
    keys = k.permute(0, 2, 3, 1).contiguous()
    vals = v.permute(0, 2, 1, 4, 3).reshape(b, kvh, n, hd)
    q = s["q"].float().view(b, t, kvh, group, hd).permute(0, 2, 3, 1, 4).reshape(b, kvh, group * t, hd)
    x = torch.matmul(q, keys).view(b, heads, t, n) * hd**-0.5
    node = torch.arange(n, device=DEV) - s["base"][:, None]  # [b, n], negative in the context
    above = _ancestors(s["parents"])
    seen = above.gather(2, node.clamp(0, t - 1)[:, None].expand(-1, t, -1)) & (node < t)[:, None]
    present = s["parents"] >= -1
    seen = torch.where((node < 0)[:, None], present[:, :, None], seen)
    x = x.masked_fill(~seen[:, None], -torch.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    x = x / x.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(x.view(b, kvh, group * t, n), vals).view(b, heads, t, hd).permute(0, 2, 1, 3)
    if s["gate"] is not None:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return o.to(s["q"].dtype).contiguous()


def _columns(s, dtype):
    """The conv's input columns of every node, oldest first: `[B, t, CONV, channels]`."""
    c, n = s["case"], s["channels"]
    b, t = c["batch"], c["nodes"]
    stored = s["conv"][s["slots"]].transpose(1, 2).to(dtype)  # [B, CONV - 1, channels]
    raw = s["proj"][..., :n].to(dtype)
    lane = torch.arange(b, device=DEV)
    out = torch.zeros(b, t, CONV, n, dtype=dtype, device=DEV)
    for i in range(t):
        p = s["parents"][:, i].long()
        above = stored if i == 0 else torch.where((p >= 0)[:, None, None], out[lane, p.clamp(min=0), 1:], stored)
        out[:, i] = torch.cat([above, raw[:, i : i + 1]], 1)
    return out


def _plain_prep(s):
    c, n = s["case"], s["channels"]
    b, t, kh, vh = c["batch"], c["nodes"], c["k_heads"], c["v_heads"]
    cols = _columns(s, torch.float64)  # the rounding below has borders, next to which 32 bits are too few
    w = s["conv_w"].double()
    acc = cols[:, :, 0] * w[:, 0]
    for j in range(1, CONV):
        acc = acc + cols[:, :, j] * w[:, j]
    y = (acc / (1.0 + torch.exp(-acc))).to(s["proj"].dtype).float()  # a tensor of the model's type
    q, k = (y[..., i * kh * KD : (i + 1) * kh * KD].view(b, t, kh, KD) for i in range(2))
    q, k = (x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) + EPS) for x in (q, k))
    x = s["proj"][..., -vh:].float() + s["dt_bias"]
    softplus = torch.where(x > 20.0, x, torch.log1p(torch.exp(x.clamp(max=20.0))))
    live = (s["parents"] >= -1)[..., None]
    out = {"q": q * KD**-0.5, "k": k, "v": y[..., 2 * kh * KD :].reshape(b, t, vh, KD),
           "g": -torch.exp(s["a_log"]) * softplus, "beta": 1.0 / (1.0 + torch.exp(-s["proj"][..., -2 * vh : -vh].float()))}
    return {name: torch.where(live if x.dim() == 3 else live[..., None], x, 0.0) for name, x in out.items()}


def _step(state, k, v, g, beta):
    state = state * torch.exp(g)[..., None, None]
    delta = (v - (state * k[..., None]).sum(-2)) * beta[..., None]
    return state + k[..., None] * delta[..., None, :]


def _plain_rule(s):
    c = s["case"]
    rep, t = c["v_heads"] // c["k_heads"], c["nodes"]
    q, k = s["q"].repeat_interleave(rep, 2), s["k"].repeat_interleave(rep, 2)
    first = s["state"][s["slots"]]
    lane = torch.arange(c["batch"], device=DEV)
    held, out = torch.empty(t, *first.shape, device=DEV), torch.zeros_like(s["v"])
    for i in range(t):
        p = s["parents"][:, i].long()
        above = first if i == 0 else torch.where((p >= 0)[:, None, None, None], held[p.clamp(min=0), lane], first)
        held[i] = _step(above, k[:, i], s["v"][:, i], s["g"][:, i], s["beta"][:, i])
        out[:, i] = (held[i] * q[:, i, :, :, None]).sum(-2) * (p >= -1)[:, None, None]
    return out


def _plain_commit(s):
    c = s["case"]
    rep = c["v_heads"] // c["k_heads"]
    lane, slots = torch.arange(c["batch"], device=DEV), s["slots"]
    state = s["state"][slots]
    window = s["conv"][slots]
    for i in range(c["longest"]):
        on, at = i < s["lengths"], s["path"][:, i]
        k = s["k"][lane, at].repeat_interleave(rep, 1)
        state = torch.where(on[:, None, None, None], _step(state, k, s["v"][lane, at], s["g"][lane, at], s["beta"][lane, at]), state)
        raw = s["proj"][lane, at, : s["channels"], None]
        window = torch.where(on[:, None, None], torch.cat([window[..., 1:], raw], -1), window)
    s["state"][slots] = state
    s["conv"][slots] = window
    return {"state": s["state"], "conv": s["conv"]}


def _plain_take(s):
    c = s["case"]
    b, t = c["batch"], c["nodes"]
    lane, node = torch.arange(b, device=DEV), torch.arange(t, device=DEV)
    at = torch.zeros(b, dtype=torch.long, device=DEV)
    going = torch.ones(b, dtype=torch.bool, device=DEV)
    n = torch.zeros(b, dtype=torch.long, device=DEV)  # accepted drafts
    path = [at]
    for i in range(1, t):
        best = s["best"][lane, at]
        fits = (s["parents"] == at[:, None]) & (s["tokens"] == best[:, None]) & (node > at[:, None])
        stop = (s["stops"] == best[:, None]).any(1)
        going = going & fits.any(1) & ~stop & (i <= s["budget"] - 1)
        at = torch.where(going, fits.int().argmax(1), at)
        n = n + going
        path.append(at)
    bonus = s["best"][lane, at]
    left = s["budget"] - n - 1
    lengths = torch.where(s["active"], n + 1, 1)
    path = torch.stack(path, 1)
    to = s["base"][:, None] + node
    of = s["base"][:, None] + torch.where(node < lengths[:, None], path, node)  # the others' rows are written as they were
    to, of = ((s["table"].gather(1, x // BLOCK).long(), x % BLOCK) for x in (to, of))
    s["k"][:, to[0] * BLOCK + to[1]] = s["k"][:, of[0] * BLOCK + of[1]]
    s["v"][:, to[0], :, :, to[1]] = s["v"][:, of[0], :, :, of[1]]
    return {"path": path, "accept_len": n, "lengths": lengths, "keep": s["active"][:, None] & (node <= n[:, None]),
            "bonus": bonus, "next_pos": s["pos"] + n + 1, "budget_left": left,
            "live": ~(s["stops"] == bonus[:, None]).any(1) & (left > 0), "hidden_src": lane * t + at, "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------- 64 bits


def _ways(parents):
    """For each node of one lane its way from the root, or None where it is absent."""
    ways = []
    for i, p in enumerate(parents.tolist()):
        ways.append(None if p < -1 or (p >= 0 and ways[p] is None) else (ways[p] if p >= 0 else []) + [i])
    return ways


def _exact_attention(s):
    c = s["case"]
    b, t, heads, hd = s["q"].shape
    group = heads // s["k_pool"].shape[1]
    out = torch.zeros(b, t, heads, hd, dtype=torch.float64, device=DEV)
    for j, base in enumerate(_bases(c)):
        key = torch.arange(base + t, device=DEV)
        block = s["table"][j].long()[key // BLOCK]
        hidden = torch.ones(t, base + t, dtype=torch.bool)
        ways = _ways(s["parents"][j])
        for i, way in enumerate(ways):
            if way is not None:
                hidden[i, :base] = False
                hidden[i, [base + x for x in way]] = False
        hidden = hidden.to(DEV)
        rows = torch.tensor([i for i, way in enumerate(ways) if way is not None], device=DEV)
        for h in range(0, heads, group):
            keys = s["k_pool"][block * BLOCK + key % BLOCK, h // group].double()
            vals = s["v_pool"][block, h // group, :, key % BLOCK].double()
            q = s["q"][j, rows, h : h + group].double()
            x = (q.reshape(-1, hd) @ keys.t()).view(len(rows), group, -1) / math.sqrt(hd)
            x = torch.softmax(x.masked_fill(hidden[rows][:, None], -torch.inf), -1)
            out[j, rows, h : h + group] = (x.view(-1, base + t) @ vals).view(len(rows), group, hd)
    return out * torch.sigmoid(s["gate"].double()) if c["gate"] else out


def _exact_prep(s):
    c, n = s["case"], s["channels"]
    b, t, kh, vh = c["batch"], c["nodes"], c["k_heads"], c["v_heads"]
    q, k = (torch.zeros(b, t, kh, KD, dtype=torch.float64, device=DEV) for _ in range(2))
    v = torch.zeros(b, t, vh, KD, dtype=torch.float64, device=DEV)
    g, beta = (torch.zeros(b, t, vh, dtype=torch.float64, device=DEV) for _ in range(2))
    for j in range(b):
        stored = s["conv"][s["slots"][j]].double()
        raw = s["proj"][j, :, :n].double()
        for i, way in enumerate(_ways(s["parents"][j])):
            if way is None:
                continue
            inputs = torch.cat([stored, raw[way].t()], 1)[:, -CONV:]
            y = torch.nn.functional.silu((inputs * s["conv_w"].double()).sum(1))
            y = y.to(s["proj"].dtype).double()
            for x, at in ((q, 0), (k, kh * KD)):
                head = y[at : at + kh * KD].view(kh, KD)
                x[j, i] = head / torch.sqrt((head * head).sum(-1, keepdim=True) + EPS)
            v[j, i] = y[2 * kh * KD :].view(vh, KD)
            beta[j, i] = torch.sigmoid(s["proj"][j, i, -2 * vh : -vh].double())
            x = s["proj"][j, i, -vh:].double() + s["dt_bias"].double()
            g[j, i] = -s["a_log"].double().exp() * torch.logaddexp(x, torch.zeros_like(x))
    return {"q": q / math.sqrt(KD), "k": k, "v": v, "g": g, "beta": beta}


def _exact_rule(s):
    """The closed form: with D(i, j) the decay from j to i and j before i on its way, the corrections u solve
    u_i = beta_i (v_i - D(i) S^T k_i - sum_j D(i, j) (k_i . k_j) u_j)."""
    c = s["case"]
    rep, t = c["v_heads"] // c["k_heads"], c["nodes"]
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device=DEV)
    for j in range(c["batch"]):
        ways = _ways(s["parents"][j])
        on = torch.zeros(t, t, dtype=torch.float64)
        for i, way in enumerate(ways):
            if way is not None:
                on[i, way] = 1.0
        on = on.to(DEV)
        q, k = (x[j].double().transpose(0, 1).repeat_interleave(rep, 0) for x in (s["q"], s["k"]))  # [heads, t, KD]
        v, state = s["v"][j].double().transpose(0, 1), s["state"][s["slots"][j]].double()
        total = on @ s["g"][j].double()  # [t, heads]
        total = total.t()
        decay = torch.exp((total[:, :, None] - total[:, None, :]).masked_fill(on == 0, -torch.inf))
        beta = s["beta"][j].double().t()[..., None]
        grown = torch.exp(total)[..., None]
        kt = k.transpose(1, 2).contiguous()
        near = decay * (k @ kt)
        u = v - grown * (k @ state)
        for i in range(t):
            if i:
                u[:, i] -= (near[:, i, :i, None] * u[:, :i]).sum(1)
            u[:, i] *= beta[:, i]
        o = grown * (q @ state) + (decay * (q @ kt)) @ u
        out[j] = (o * on.diagonal()[:, None]).transpose(0, 1)
    return out


def _exact_commit(s):
    c = s["case"]
    rep = c["v_heads"] // c["k_heads"]
    state, conv = s["state"].double(), s["conv"].double()
    for j, n in enumerate(_lengths(c)):
        slot, way = int(s["slots"][j]), s["path"][j, :n].tolist()
        for i in way:
            k, v, beta = s["k"][j, i].double().repeat_interleave(rep, 0), s["v"][j, i].double(), s["beta"][j, i].double()
            m = state[slot] * s["g"][j, i].double().exp()[:, None, None]
            u = beta[:, None] * (v - (k[:, None] @ m)[:, 0])
            state[slot] = m + k[:, :, None] @ u[:, None, :]
        rows = s["proj"][j, way, : s["channels"]].double().t()
        conv[slot] = torch.cat([conv[slot], rows], 1)[:, -(CONV - 1) :]
    return {"state": state, "conv": conv}


def _exact_take(s):
    c = s["case"]
    t, k, v = c["nodes"], s["k"].double(), s["v"].double()
    told = {name: [] for name in ("path", "accept_len", "lengths", "keep", "bonus", "next_pos", "budget_left", "live", "hidden_src")}
    parents, tokens, best, stops, table = (s[x].tolist() for x in ("parents", "tokens", "best", "stops", "table"))
    for j, base in enumerate(_bases(c)):
        way, budget = [0], int(s["budget"][j])
        while len(way) < budget and best[j][way[-1]] not in stops[j]:
            below = [i for i in range(way[-1] + 1, t) if parents[j][i] == way[-1] and tokens[j][i] == best[j][way[-1]]]
            if not below:
                break
            way.append(below[0])
        active = j % 11 != 10
        if active and len(way) > 1:
            of, to = (base + torch.tensor(x, device=DEV) for x in (way, range(len(way))))
            of, to = ((torch.tensor(table[j], device=DEV)[x // BLOCK], x % BLOCK) for x in (of, to))
            k[:, to[0] * BLOCK + to[1]] = k[:, of[0] * BLOCK + of[1]].clone()
            v[:, to[0], :, :, to[1]] = v[:, of[0], :, :, of[1]].clone()
        n, bonus = len(way) - 1, best[j][way[-1]]
        for name, x in (("path", way + [way[-1]] * (t - len(way))), ("accept_len", n), ("lengths", n + 1 if active else 1),
                        ("keep", [active and i <= n for i in range(t)]), ("bonus", bonus), ("next_pos", base + n + 1),
                        ("budget_left", budget - n - 1), ("live", bonus not in stops[j] and budget > n + 1),
                        ("hidden_src", j * t + way[-1])):
            told[name].append(x)
    return {**{name: torch.tensor(x, device=DEV) for name, x in told.items()}, "k": k, "v": v}


def exact(case, seed):
    return globals()[f"_exact_{case['kind']}"](prepare(case, seed))


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    c = case
    rows = sum(_sizes(c))
    if c["kind"] == "attention":  # every live node sees its context and at least itself
        heads, kvh = LAYOUTS[c["head_dim"]]
        pairs = sum(n * (base + 1) for n, base in zip(_sizes(c), _bases(c)))
        keys = sum(n + base for n, base in zip(_sizes(c), _bases(c)))
        moved = rows * heads * (3 if c["gate"] else 2) + 2 * keys * kvh
        return {"bytes": 2 * c["head_dim"] * moved, "flops": 4 * c["head_dim"] * heads * pairs}
    if c["kind"] == "take":  # the rows that change their place, read once and written once
        kvh = LAYOUTS[c["head_dim"]][1]
        moved = sum(min(n, 2 if j % 7 == 3 else n) - 1 for j, n in enumerate(_lengths(c)) if j % 11 != 10)
        return {"bytes": 2 * 2 * 2 * c["layers"] * moved * kvh * c["head_dim"] + 28 * c["batch"] * c["nodes"], "flops": 0}
    kh, vh = c["k_heads"], c["v_heads"]
    if c["kind"] == "prep":
        n, width = (2 * kh + vh) * KD, 4 if c["dtype"] == "f32" else 2
        return {"bytes": rows * ((n + 2 * vh) * width + 4 * (n + 2 * vh)) + c["batch"] * n * (CONV - 1) * width,
                "flops": rows * n * (2 * CONV + 4)}
    if c["kind"] == "rule":  # S^T k and S^T q of every node, and the update that its children see
        return {"bytes": 4 * (c["batch"] * vh * KD * KD + rows * (2 * kh * KD + 2 * vh * KD + 2 * vh)),
                "flops": 4 * rows * vh * KD * KD}
    steps = sum(_lengths(c))
    width = 4 if c["dtype"] == "f32" else 2
    return {"bytes": 4 * (2 * c["batch"] * vh * KD * KD + steps * (kh * KD + vh * KD + 2 * vh))
            + width * (2 * kh + vh) * KD * c["batch"] * 2 * (CONV - 1), "flops": 6 * steps * vh * KD * KD}
