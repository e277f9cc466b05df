"""Launches of the tree's operators that would reach 2^32 threads, refused at the C entry points before anything is launched."""

from __future__ import annotations

import pytest
import torch

import _mtpk
from tests.test_tree_cpu import PAIR, P, lib  # noqa: F401


def _rule(lib, rows: int, heads: int, qk: int, vd: int, t: int = 1, base: int = P) -> int:  # noqa: F811
    return lib.mtpk_delta_rule_tree(base, 1, base, rows, t, heads, qk, 16, vd, base, base, base, base, base, base, _mtpk.I32, PAIR, base, None)


# rows, heads, q/k heads, v_dim, nodes: workgroups x threads
TOO_MANY = [
    (1 << 20, 16, 16, 16, 1),  # 2^24 of 256
    (1 << 22, 16, 16, 16, 16),  # 2^26 of 256
    ((1 << 20) + 4096, 16, 16, 64, 40),
    (1 << 23, 5, 1, 4, 1),  # five units a q/k head: 2^24 of 256
    (1 << 24, 4, 1, 64, 33),  # 2^24 of 256, at most a workgroup a compute unit
    (1 << 20, 64, 4, 64, 64),  # 2^24 of 256 or 2^23 of 512
]
# the same shapes, a workgroup below
FITTING = [(((1 << 20) - 1), 16, 16, 16, 1), ((1 << 23) - 1, 5, 1, 4, 1), ((1 << 20) - 1, 64, 4, 64, 64)]


@pytest.mark.parametrize("rows,heads,qk,vd,t", TOO_MANY)
def test_rules_of_too_many_threads_are_refused(lib, rows, heads, qk, vd, t) -> None:  # noqa: F811
    assert _rule(lib, rows, heads, qk, vd, t) == _mtpk.EINVAL


@pytest.mark.parametrize("rows,heads,qk,vd", [(1 << 22, 16, 16, 16), (1 << 22, 16, 16, 3)])
def test_step_by_step_rules_of_too_many_threads_are_refused(lib, rows, heads, qk, vd) -> None:  # noqa: F811
    """Operands off 16 bytes, or a v_dim that is no multiple of 4: workgroups of 64 threads."""
    assert _rule(lib, rows, heads, qk, vd, base=P + 4) == _mtpk.EINVAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="the call would be launched, on addresses of nothing")
@pytest.mark.parametrize("rows,heads,qk,vd,t", FITTING)
def test_rules_below_the_limit_reach_the_launch(lib, rows, heads, qk, vd, t) -> None:  # noqa: F811
    assert _rule(lib, rows, heads, qk, vd, t) not in (0, _mtpk.EINVAL)  # no device here
