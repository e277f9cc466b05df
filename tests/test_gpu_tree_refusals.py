"""What the operators of a tree refuse, checked on the host before anything is launched."""

from __future__ import annotations

import pytest
import torch

import attention
import deltanet
import graph_mtp

pytestmark = pytest.mark.gpu


def refused(call, good: dict, bad: list[dict]) -> None:
    call(**good)
    for change in bad:
        with pytest.raises(ValueError):
            call(**{**good, **change})


def trees(dev, b: int, t: int, dtype=torch.int32) -> torch.Tensor:
    return torch.arange(-1, t - 1, device=dev).to(dtype).expand(b, t)


PARENTS = [lambda d: trees(d, 2, 3), lambda d: trees(d, 1, 4), lambda d: trees(d, 2, 4).float(), lambda d: trees("cpu", 2, 4),
           lambda d: trees(d, 2, 4, torch.int16), lambda d: trees(d, 2, 4)[0]]


def test_attention(dev) -> None:
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    good = {"q": z(2, 4, 4, 64), "k_pool": z(64, 2, 64), "v_pool": z(4, 2, 64, 16), "block_table": z(2, 2, dtype=torch.int32),
            "base_pos": z(2, dtype=torch.int64), "ctx_len": 32, "scale": 0.1, "parents": trees(dev, 2, 4), "gate": z(2, 4, 4, 64)}
    refused(attention.paged_attention_tree, good, [
        *({"parents": p(dev)} for p in PARENTS), {"q": z(2, 65, 4, 64), "parents": trees(dev, 2, 65), "gate": None}, {"q": z(2, 4, 4, 64).float()},
        {"q": z(2, 0, 4, 64), "parents": trees(dev, 2, 0), "gate": None}, {"q": z(2, 4, 4, 96), "gate": None}, {"q": z(2, 4, 3, 64), "gate": None},
        {"q": z(2, 4, 4, 64).cpu()}, {"gate": z(2, 4, 4, 32)}, {"gate": z(2, 4, 4, 64).float()}, {"gate": z(2, 4, 4, 64).cpu()}, {"ctx_len": 33},
        {"ctx_len": -1}, {"scale": 0.0}, {"scale": float("nan")}, {"scale": -1.0}, {"k_pool": z(63, 2, 64)}, {"k_pool": z(64, 2, 128)},
        {"v_pool": z(4, 2, 64, 8)}, {"v_pool": z(4, 2, 64, 16).cpu()}, {"block_table": z(1, 2, dtype=torch.int32)}, {"base_pos": z(3, dtype=torch.int64)},
        {"base_pos": z(2, dtype=torch.float32)},
    ])  # fmt: skip


def test_prep(dev) -> None:
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    width = 2 * 16 + 2 * 16
    good = {"proj": z(2, 4, width + 2 * 16 + 4), "conv_state": z(3, width, 3), "slots": z(2, dtype=torch.int64), "conv_w": z(width, 4),
            "a_log": z(2, dtype=torch.float32), "dt_bias": z(2, dtype=torch.float32), "k_heads": 1, "k_dim": 16, "v_heads": 2, "v_dim": 16,
            "parents": trees(dev, 2, 4)}
    refused(deltanet.prep_tree, good, [
        *({"parents": p(dev)} for p in PARENTS), {"proj": z(2, 4, width + 2 * 16 + 3)}, {"proj": z(2, 4, 100).half()}, {"proj": good["proj"][0]},
        {"proj": z(2, 4, 100).cpu()}, {"proj": z(2, 4, 100, dtype=torch.float32)}, {"conv_state": z(3, width, 2)}, {"conv_state": z(0, width, 3)},
        {"conv_state": z(3, 3, width).transpose(1, 2)}, {"conv_w": z(width, 10), "conv_state": z(3, width, 9)}, {"conv_w": z(width, 1)},
        {"conv_w": z(width, 4).cpu()}, {"slots": z(3, dtype=torch.int64)}, {"slots": z(2, dtype=torch.float32)}, {"a_log": z(3)},
        {"dt_bias": z(2, dtype=torch.int32)}, {"k_heads": 0}, {"k_dim": 257}, {"v_dim": 0},
        {"proj": z(2, 65, 100), "parents": trees(dev, 2, 65)},
    ])  # fmt: skip


def test_rule_and_commit(dev) -> None:
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    rows = {"k": z(2, 4, 1, 16), "v": z(2, 4, 2, 8), "g": z(2, 4, 2), "beta": z(2, 4, 2)}
    bad_rows = [{"k": z(2, 4, 3, 16)}, {"k": z(2, 4, 1, 8)}, {"v": z(2, 4, 2, 9)}, {"v": z(2, 3, 2, 8)}, {"g": z(2, 4)}, {"beta": z(1, 4, 2)},
                {"beta": z(2, 4, 2).cpu()}, {"g": z(2, 4, 2, dtype=torch.int32)}]
    state = z(3, 2, 16, 8)
    bad_states = [z(3, 2, 24, 8), z(3, 2, 16, 8).half(), z(3, 2, 8, 16).transpose(2, 3), state[0], z(3, 2, 16, 8).cpu()]
    good = {"state": state, "slots": z(2, dtype=torch.int64), "q": z(2, 4, 1, 16), **rows, "parents": trees(dev, 2, 4)}
    refused(deltanet.delta_rule_tree, good, [
        *({"parents": p(dev)} for p in PARENTS), *bad_rows, *({"state": s} for s in bad_states), {"q": z(2, 4, 2, 16)}, {"slots": z(3, dtype=torch.int64)},
        {"slots": None, "state": z(1, 2, 16, 8)}, {"slots": z(2)},
    ])  # fmt: skip
    long = lambda *s: z(*s, dtype=torch.int64)  # noqa: E731
    good = {"state": state, "conv_state": z(3, 32, 3), "slots": torch.tensor([0, 2], device=dev), **rows, "path": long(2, 4),
            "lengths": torch.ones(2, dtype=torch.int64, device=dev), "proj": z(2, 4, 50), "channels": 32}
    refused(deltanet.commit_path, good, [
        *bad_rows, *({"state": s} for s in bad_states), {"path": long(2, 3)}, {"path": z(2, 4)}, {"lengths": long(3)}, {"slots": z(2)},
        {"proj": z(2, 4, 31)}, {"proj": z(2, 3, 50)}, {"proj": z(2, 4, 50).bfloat16()}, {"channels": 31}, {"channels": 0}, {"conv_state": z(3, 32, 9)},
        {"conv_state": z(3, 3, 32).transpose(1, 2)}, {"conv_state": z(3, 32, 3).cpu()}, {"path": long(2, 4).cpu()},
    ])  # fmt: skip


def test_acceptance_and_kept_rows(dev) -> None:
    long = lambda *s: torch.zeros(*s, dtype=torch.int64, device=dev)  # noqa: E731
    good = {"step_argmax": long(2, 4), "tokens": long(2, 4), "parents": trees(dev, 2, 4), "active": long(2).bool(), "pos": long(2),
            "budget": long(2), "stops": long(2, 3)}
    refused(graph_mtp.tree_accept, good, [
        *({"parents": p(dev)} for p in PARENTS), {"tokens": long(2, 3)}, {"tokens": long(2, 4).int()}, {"step_argmax": long(2, 4).int()},
        {"active": long(2)}, {"active": long(3).bool()}, {"pos": long(3)}, {"budget": long(2, 1)}, {"stops": long(3)}, {"stops": long(1, 3)},
        {"stops": long(2, 3).int()}, {"tokens": long(2, 4).cpu()}, {"step_argmax": long(2, 65), "tokens": long(2, 65), "parents": trees(dev, 2, 65)},
    ])  # fmt: skip
    k, v = torch.zeros(48, 2, 8, device=dev), torch.zeros(3, 2, 8, 16, device=dev)
    good = {"pools": [k, v], "block_table": long(2, 1).int(), "base_pos": long(2), "path": long(2, 4), "lengths": long(2)}
    refused(attention.keep_path, good, [
        {"pools": []}, {"pools": [k, v.cpu()]}, {"pools": [k[:47]]}, {"pools": [k, torch.zeros(4, 2, 8, 16, device=dev)]},
        {"pools": [k.double(), v.double()]}, {"pools": [torch.zeros(48, 1, 2, device=dev)]}, {"pools": [k.transpose(1, 2)]},
        {"block_table": long(1, 1)}, {"block_table": long(2, 0)}, {"block_table": long(2, 1).float()}, {"block_table": long(2, 1).cpu()},
        {"path": long(2, 65)}, {"path": long(2, 0)}, {"path": long(4)}, {"lengths": long(3)}, {"base_pos": long(2).float()},
        {"lengths": long(2).cpu()},
    ])  # fmt: skip
