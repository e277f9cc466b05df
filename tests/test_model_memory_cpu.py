"""What the CPU forward holds on to."""

from __future__ import annotations

import weakref

import torch

import verify_model as vm
from tests import model_helpers as mh


def test_a_chain_holds_no_states_it_has_left(monkeypatch) -> None:
    """The rule's states of a chain die as the next ones are made."""
    model, t, alive = mh.build(), 24, []
    step = vm.delta_rule_step
    held: list[int] = []

    def counted(state, *args):
        if not alive:
            alive.append(weakref.ref(state))  # the stored one
        new, out = step(state, *args)
        alive.append(weakref.ref(new))
        held.append(sum(r() is not None for r in alive))
        return new, out

    monkeypatch.setattr(vm, "delta_rule_step", counted)
    i = model.cfg.layer_types.index(vm.DELTANET)
    h = torch.randn(1, t, model.cfg.hidden, generator=torch.Generator().manual_seed(0))
    model.deltanet_verify(model.layers[i], model.pool[i], h, torch.tensor([0]))
    assert len(held) == t and max(held) <= 2
