"""The half-precision network's training step without a GPU: which parameters go to which optimizer."""

from __future__ import annotations

import pytest

from create_graph_b200.half_mlp import HalfMLPModel, Trainer
from create_graph_b200.mlp import MLPSpec
from create_graph_b200.optim import FusedAdamW, FusedMuon


@pytest.mark.parametrize("depth", [1, 2, 4])
def test_optimizers_of_each_depth(depth):
    model = HalfMLPModel(MLPSpec(hidden=16), depth=depth)
    trainer = Trainer(model)
    matrices = {id(layer.weight) for layer in model.network.rest}
    assert len(matrices) == depth - 1
    groups = {type(o): {id(p) for p in o.grads.params} for o in trainer.optimizers}
    assert groups.get(FusedMuon, set()) == matrices
    assert groups[FusedAdamW] == {id(p) for p in model.parameters()} - matrices
    assert [o.grads for o in trainer.optimizers] == trainer.grads
