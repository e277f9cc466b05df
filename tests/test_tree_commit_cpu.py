"""Which entries of a path a commit takes on the CPU: as on the device, those before the first that is no node, at most `lengths`."""

from __future__ import annotations

import pytest
import torch

from tests import model_helpers as mh
from tests import tree_inputs


def committed(path: list[list[int]], lengths: list[int]) -> list[torch.Tensor]:
    model = mh.build()
    for lane, p in enumerate(mh.prompts()):
        model.prefill(lane, p)
    model.blocks.grow_many([0, 1], [22, 22])
    pos, tree = torch.tensor([16, 16]), tree_inputs.batch(["random", "star"], 6)
    res = model.forward_rows(torch.tensor(mh.prompts(2, 6, seed=3)), [0, 1], pos, 22, parents=tree)
    model.commit_path(res, [0, 1], pos, torch.tensor(path), torch.tensor(lengths))
    return [x for lane in range(2) for x in mh.slot_state(model, lane, 16)]


@pytest.mark.parametrize("path,lengths,like", [
    ([[0, 1, -1, -1, -1, -1], [0, 6, 6, 6, 6, 6]], [6, 6], [2, 1]),  # no node ends a path
    ([[0, 2**40, 1, 2, 3, 4], [0, 3, 3, -(2**40), 1, 1]], [4, 2], [1, 2]),
    ([[0, 1, 2, 3, 4, 5], [-1, 0, 0, 0, 0, 0]], [2**40, -3], [6, 0]),
])
def test_where_a_path_ends(path, lengths, like) -> None:
    got = committed(path, lengths)
    want = committed([[s if 0 <= s < 6 else 0 for s in p] for p in path], like)
    assert all(torch.equal(x, y) for x, y in zip(got, want, strict=True))
