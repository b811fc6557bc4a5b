"""
The half-precision energy network (create_graph_b200.half_mlp): one
conservative-force step against float64 eager torch, and training with Muon and
AdamW together.

Tolerances, norm-wise relative, u = 2^-11 (fp16): a layer's output passes
through about four roundings (operands, weights, bias, output), so energies are
within 4 u per layer; forces add the backward products and gz (8 u per layer);
the parameter gradient goes through both passes (16 u per layer). Three layers;
the fp32 readout adds 1e-5 (fp32 GEMM precision).
"""

from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

import create_graph_b200 as cg
from create_graph_b200 import native
from create_graph_b200 import nn as cgnn
from create_graph_b200.gemm import gemm_precision
from create_graph_b200.half_mlp import HalfMLPModel, Trainer
from create_graph_b200.mlp import MLPSpec, molecules_csr, synthetic_batch

pytestmark = pytest.mark.gpu
U = 2.0**-11
DEPTH = 3


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


def setup(spec, dtype, seed=0):
    torch.manual_seed(seed)
    model = HalfMLPModel(spec, depth=DEPTH, dtype=dtype).cuda()
    pos, e, f = (t.cuda() for t in synthetic_batch(spec, seed=seed))
    return model, {"pos": pos, "molecules": molecules_csr(spec, "cuda")}, e, f


def reference(model, spec, pos, e_target, f_target):
    """(energy, forces, loss, gradients) of the same network in float64 on the CPU."""
    params = {name: p.detach().double().cpu().requires_grad_(True) for name, p in model.named_parameters()
              if name.startswith("network.")}
    pos = pos.detach().double().cpu().requires_grad_(True)
    x = pos.view(spec.n_mol, spec.n_atom, 3)
    h = (x - x.mean(dim=1, keepdim=True)).reshape(-1, 3)
    h = F.silu(F.linear(h, params["network.first.weight"], params["network.first.bias"]))
    for i in range(DEPTH - 1):
        h = h + F.gelu(F.linear(h, params[f"network.rest.{i}.weight"], params[f"network.rest.{i}.bias"]))
    e = F.linear(h, params["network.readout.weight"], params["network.readout.bias"]).view(spec.n_mol, -1).sum(1)
    (g,) = torch.autograd.grad(e.sum(), pos, create_graph=True)
    loss = (e - e_target.double().cpu()).square().mean() + (-g - f_target.double().cpu()).square().mean()
    return e, -g, loss, dict(zip(params, torch.autograd.grad(loss, list(params.values()))))


@pytest.mark.parametrize("spec", [MLPSpec(), MLPSpec(n_mol=3, n_atom=17, hidden=72)])
def test_step_against_float64(spec):
    model, batch, e_target, f_target = setup(spec, torch.float16)
    with gemm_precision("fp32"):
        out, grads = cg.create_graph(model, batch)
        loss = cgnn.energy_force_loss(out["energy"], grads["pos"], e_target, f_target)
        loss.backward()
    e, f, want, want_grads = reference(model, spec, batch["pos"], e_target, f_target)
    assert rel(out["energy"], e) < 4 * DEPTH * U + 1e-5
    assert rel(-grads["pos"], f) < 8 * DEPTH * U + 1e-5
    assert rel(loss, want) < 16 * DEPTH * U
    named = dict(model.named_parameters())
    for name, g in want_grads.items():
        if float(g.norm()) > 0.0:
            assert named[name].grad.dtype == torch.float32
            assert rel(named[name].grad, g) < 16 * DEPTH * U + 1e-5, name
    assert native.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_training_lowers_the_loss_and_repeats(dtype):
    def run():
        model, batch, e_target, f_target = setup(MLPSpec(), dtype, seed=1)
        trainer = Trainer(model, lr=5e-3)
        return torch.stack([trainer.step(batch, e_target, f_target) for _ in range(60)]), model

    losses, model = run()
    again, other = run()
    assert float(losses[-1]) < 0.7 * float(losses[0])
    assert torch.equal(losses, again)
    assert all(torch.equal(a, b) for a, b in zip(model.parameters(), other.parameters()))
