"""
Half-precision layers inside checkpointed blocks: one conservative-force step of
HalfMLPModel whose hidden layers are recomputed, at every tier of the memory
budget, against the same network in float64 and against the step that keeps
everything.

Tolerances as in test_half_mlp_gpu.py (u = 2^-11, three layers): energies 4 u a
layer, forces 8 u, parameter gradients 16 u. A recompute runs the same kernels on
the same inputs, so energies and forces equal those of the kept step bit for bit;
the deferred parameter backward sums in another order.
"""

from __future__ import annotations

import pytest
import torch

import create_graph_b200 as cg
from create_graph_b200 import native
from create_graph_b200 import nn as cgnn
from create_graph_b200.gemm import gemm_precision
from create_graph_b200.half_mlp import HalfMLPModel
from create_graph_b200.mlp import MLPSpec, molecules_csr, synthetic_batch
from tests.test_half_mlp_gpu import DEPTH, U, reference, rel

pytestmark = pytest.mark.gpu
SPEC = MLPSpec(n_mol=3, n_atom=17, hidden=72)


def step(config):
    torch.manual_seed(0)
    model = HalfMLPModel(SPEC, depth=DEPTH, dtype=torch.float16, config=config).cuda()
    pos, e, f = (t.cuda() for t in synthetic_batch(SPEC, seed=0))
    batch = {"pos": pos, "molecules": molecules_csr(SPEC, "cuda")}
    with gemm_precision("fp32"):
        out, grads = cg.create_graph(model, batch)
        loss = cgnn.energy_force_loss(out["energy"], grads["pos"], e, f)
        loss.backward()
    return model, batch, (e, f), out["energy"], grads["pos"]


@pytest.mark.parametrize("blocks", [r"rest\.\d+", r"first|rest\.\d+"])
@pytest.mark.parametrize("budget", [None, 0.5, 0.25])
@pytest.mark.parametrize("backend", ["inductor", "eager"])
def test_checkpointed_layers(backend, budget, blocks):
    _, _, _, kept_energy, kept_grad = step(None)
    config = cg.CompileConfig(backend=backend, checkpoint=blocks, memory_budget=budget)
    model, batch, targets, energy, grad = step(config)
    assert torch.equal(energy, kept_energy) and torch.equal(grad, kept_grad)
    e, f, _, want = reference(model, SPEC, batch["pos"], *targets)
    assert rel(energy, e) < 4 * DEPTH * U + 1e-5
    assert rel(-grad, f) < 8 * DEPTH * U + 1e-5
    named = dict(model.named_parameters())
    for name, g in want.items():
        if float(g.norm()) > 0.0:
            assert rel(named[name].grad, g) < 16 * DEPTH * U + 1e-5, name
    assert native.device_error() == 0
