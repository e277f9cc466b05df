"""Acceptance where node 0 is absent: what hangs below an absent node is absent too, so nothing is accepted."""

from __future__ import annotations

import pytest
import torch

import graph_mtp
from oracle import tree_ref

# node 0 of lanes 0, 1, 3, 4 is no node; lane 2 is whole; on every lane the model agrees with every token
PARENTS = [[-2, 0, 1, 2], [0, 0, 1, 2], [-1, 0, 1, 2], [2**31 - 1, 0, 0, 1], [-(2**31), -1, 0, 1]]


def call(device: str, dtype: torch.dtype) -> graph_mtp.TreeAccept:
    b, t = len(PARENTS), 4
    ones = torch.ones(b, t, dtype=torch.long)
    args = (ones, ones, torch.tensor(PARENTS, dtype=dtype), torch.tensor([True, True, True, True, False]), torch.arange(b),
            torch.full((b,), 9), torch.full((b, 2), -1))
    return graph_mtp.tree_accept(*(x.to(device) for x in args))


def check(got: graph_mtp.TreeAccept) -> None:
    assert got.accept_len.tolist() == [0, 0, 3, 0, 0]
    assert got.lengths.tolist() == [1, 1, 4, 1, 1]
    assert got.path.tolist() == [[0] * 4, [0] * 4, [0, 1, 2, 3], [0] * 4, [0] * 4]
    assert got.keep.tolist() == [[True] + [False] * 3, [True] + [False] * 3, [True] * 4, [True] + [False] * 3, [False] * 4]
    assert got.hidden_src.tolist() == [0, 4, 11, 12, 16] and got.next_pos.tolist() == [1, 2, 6, 4, 5]
    b = len(PARENTS)
    want = tree_ref.accept([[1] * 4] * b, [[1] * 4] * b, PARENTS, [True] * 4 + [False], list(range(b)), [9] * b, [[-1, -1]] * b)
    for name, value in want.items():
        assert getattr(got, name).tolist() == value, name


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_on_the_cpu(dtype) -> None:
    check(call("cpu", dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_on_the_device(dev, dtype) -> None:
    check(call(dev, dtype))
