"""
The half-precision dense layer and the matrix optimizer in one training step: a
per-atom energy network in bf16 or fp16, trained on energies and forces.

    molecules of n_atom atoms (synthetic_batch of create_graph_b200.mlp), centred
    region:  h = silu(x W1^T + b1)                     (half precision)
             h = h + gelu(h Wi^T + bi), i = 2 .. depth (half precision)
             e = h w^T + b                             (fp32)
             E_mol = segment sum of e over the molecule's atoms
    loss:    MSE(E, targets) + MSE(F = -dE/dpos, targets)
    update:  FusedMuon on the hidden matrices, FusedAdamW on everything else

Parameters, gradients, optimizer states, energies and the loss are fp32; the
hidden layers' operands and activations are half precision (dense.Linear), and
their products accumulate in fp32. The force pass differentiates the layers once
and the parameter backward differentiates it again, as for the fp32 layers.
"""

from __future__ import annotations

import torch
from torch import Tensor, nn

import create_graph_b200 as cg
from create_graph_b200 import dense
from create_graph_b200 import nn as cgnn
from create_graph_b200.ddp import FlatGradients
from create_graph_b200.mlp import MLPSpec
from create_graph_b200.optim import FusedAdamW, FusedMuon


class HalfEnergyMLP(nn.Module):
    """Per-atom energies summed per molecule: the cg.compile region."""

    def __init__(self, hidden: int = 64, depth: int = 3, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.dtype = dtype
        self.first = dense.Linear(3, hidden, activation="silu", dtype=dtype)
        self.rest = nn.ModuleList(
            dense.Linear(hidden, hidden, activation="gelu", dtype=dtype) for _ in range(depth - 1))
        self.readout = cgnn.Linear(hidden, 1)

    def forward(self, x: Tensor, molecules: cgnn.Csr) -> Tensor:
        h = self.first(x.to(self.dtype))
        for layer in self.rest:
            h = layer(h, residual=h)
        return cgnn.SegmentSum.apply(self.readout(h.float()), molecules).view(-1)


class HalfMLPModel(nn.Module):
    """Centring (eager) then the region."""

    def __init__(self, spec: MLPSpec = MLPSpec(), depth: int = 3, dtype: torch.dtype = torch.bfloat16,
                 config: cg.CompileConfig | None = None):
        super().__init__()
        self.spec = spec
        self.network = HalfEnergyMLP(spec.hidden, depth, dtype)
        self.region = cg.compile(self.network, config=config)

    def forward(self, batch: dict) -> dict:
        s = self.spec
        pos = batch["pos"].view(s.n_mol, s.n_atom, 3)
        centred = (pos - pos.mean(dim=1, keepdim=True)).view(s.n_mol * s.n_atom, 3)
        return {"energy": self.region(centred, batch["molecules"])}


class Trainer:
    """The training step: gradients, then one Muon update of the hidden matrices
    (a network of one layer has none) and one AdamW update of the rest, each over
    its own flat buffers."""

    def __init__(self, model: HalfMLPModel, world: int | None = None, lr: float = 1e-2):
        matrices = [layer.weight for layer in model.network.rest]
        kept = {id(p) for p in matrices}
        others = [p for p in model.parameters() if id(p) not in kept]
        self.model = model
        groups = [(make, params) for make, params in ((FusedMuon, matrices), (FusedAdamW, others)) if params]
        self.grads = [FlatGradients(params, world) for _, params in groups]
        self.optimizers = [make(grads, lr=lr) for (make, _), grads in zip(groups, self.grads)]

    def step(self, batch: dict, e_target: Tensor, f_target: Tensor) -> Tensor:
        for g in self.grads:
            g.zero()
        out, grads = cg.create_graph(self.model, batch)
        loss = cgnn.energy_force_loss(out["energy"], grads["pos"], e_target, f_target)
        loss.backward()
        for g in self.grads:
            g.allreduce()
        for optimizer in self.optimizers:
            optimizer.step()
        return loss.detach()
