"""
newton_schulz and FusedMuon at the ends of their range: norms near the smallest
and largest numbers, an eps that small, matrices of zeros. Shapes on both sides
of the size that one cluster holds (128 by 1024), and the tolerances of
test_muon_gpu.py: 1e-5 norm-wise in fp32, one rounding more in half precision.
"""

from __future__ import annotations

import pytest
import torch

from create_graph_b200 import native
from create_graph_b200.ddp import FlatGradients
from create_graph_b200.optim import NS_COEFFICIENTS, FusedMuon, newton_schulz

pytestmark = pytest.mark.gpu
SHAPES = [(40, 56), (100, 700), (150, 210), (300, 130)]


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


def orthogonalised(x, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """In float64, with eps as the fp32 number the kernels take."""
    a, b, c = coefficients
    x = x.detach().double()
    x = x / x.norm(dim=(-2, -1), keepdim=True).clamp_min(float(torch.tensor(eps, dtype=torch.float32)))
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            g = x @ x.mT
            x = a * x + (b * g + c * g @ g) @ x
        else:
            g = x.mT @ x
            x = a * x + x @ (b * g + c * g @ g)
    return x


def random(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("shape", SHAPES)
def test_smallest_eps(shape):
    x = random(*shape, seed=1)
    for eps in (1e-30, 1e-36, 1e-38, 1e-44):
        stack = torch.stack([x, torch.zeros_like(x), x * 2.0**-124, x * 2.0**-140])
        got = newton_schulz(stack, eps=eps)
        assert not got[1].any()
        # the scaled matrices keep what fp32's denormal numbers left of them
        assert rel(got, orthogonalised(stack, eps=eps)) < 1e-5
    assert native.device_error() == 0


@pytest.mark.parametrize("shape", SHAPES)
def test_largest_norms(shape):
    x = random(*shape, seed=2)
    want = newton_schulz(x)
    assert torch.equal(newton_schulz(x * 2.0**100), want)
    x = x.clamp(-1.0, 1.0) * torch.finfo(torch.float32).max
    assert rel(newton_schulz(x), orthogonalised(x)) < 1e-5


@pytest.mark.parametrize("shape", SHAPES)
def test_muon_step_on_zero_gradients(shape):
    w = random(*shape, seed=3)
    p = torch.nn.Parameter(w.clone())
    opt = FusedMuon(FlatGradients([p], None), lr=0.5, weight_decay=0.5, eps=1e-38)
    opt.step()
    assert torch.equal(p.detach(), w * 0.75)
