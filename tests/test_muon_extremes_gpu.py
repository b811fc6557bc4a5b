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


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 2.0**-8 + 1e-5)])
@pytest.mark.parametrize("coefficients,steps", [((18.0, 0.0, 0.0), 2), ((18.0, 0.0, 0.0), 3), ((17.0, -20.0, 4.0), 2),
                                                ((4.5, -4.0, 3.0), 2), ((-20.0, 3.0, 0.0), 2)])
@pytest.mark.parametrize("shape", [(1, 1), *SHAPES])
def test_coefficients_that_let_the_iteration_grow(shape, coefficients, steps, dtype, tol):
    """X, A or B beyond 16: a matrix of one direction, whose singular value is 1, and a
    random one. To first order, along that direction's path from s = 1: the polynomial
    p multiplies a relative error by |s p'(s) / p(s)|, and a step adds 2^-22 for every
    factor of its terms a X, b X X' X and c X X' X X' X, relative to p(s)."""
    a, b, c = coefficients
    s, error = 1.0, 2.0**-22
    for _ in range(steps):
        p = a * s + b * s**3 + c * s**5
        factors = abs(a * s) + 3 * abs(b * s**3) + 5 * abs(c * s**5)
        error = abs(s * (a + 3 * b * s**2 + 5 * c * s**4) / p) * error + factors / abs(p) * 2.0**-22
        s = p
    one = random(shape[0], 1, seed=4) @ random(1, shape[1], seed=5)
    for x, e in ((one, error), (random(*shape, seed=6), error if min(shape) == 1 else 0.0)):
        x = x.to(dtype)
        got = newton_schulz(x, steps=steps, coefficients=coefficients)
        assert rel(got, orthogonalised(x, steps, coefficients)) < tol + e
