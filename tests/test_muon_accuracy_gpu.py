"""
The error of fp32 newton_schulz beside that of the same iteration in torch's
fp32 products, over spectra that stress A A in different ways: Gaussian and
gradient-like matrices (off-diagonal terms of either sign under a large
diagonal), orthogonal rows (no off-diagonal terms: nothing is truncated, so
nothing may be put back) and block-diagonal grams.

Bound: 1.5 times torch's error, and 1e-6 for the planes. Each step rounds X, A
and B to pairs of fp16 planes (22 bits, 2^-23 a value); fifteen such roundings,
independent, and weighted by up to 2 on the way through the remaining steps, are
2 sqrt(15) 2^-23 = 0.9e-6.
"""

from __future__ import annotations

import pytest
import torch

from create_graph_b200 import native
from create_graph_b200.optim import NS_COEFFICIENTS, newton_schulz

pytestmark = pytest.mark.gpu
# on both sides of the size that one cluster holds (128 by 1024)
SHAPES = [(37, 2949), (55, 2364), (129, 140), (257, 1031), (1031, 260), (512, 512), (55, 600), (600, 55), (90, 1000),
          (128, 128), (46, 200), (20, 16)]


def draw(*shape, gen, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, dtype=dtype)


def gaussian(r, c, gen):
    return draw(r, c, gen=gen)


def gradient(r, c, gen):
    k = max(1, min(32, r // 2, c // 2))
    return 1e-3 * (draw(r, k, gen=gen) @ draw(k, c, gen=gen) / k**0.5 + draw(r, c, gen=gen))


def orthogonal(r, c, gen):
    q = torch.linalg.qr(draw(max(r, c), min(r, c), gen=gen, dtype=torch.float64))[0]
    return (q if r >= c else q.t()).float().contiguous()


def blocks(r, c, gen):
    x = torch.zeros(r, c)
    for i in range(8):
        rows, cols = (slice(i * n // 8, (i + 1) * n // 8) for n in (r, c))
        x[rows, cols] = draw(rows.stop - rows.start, cols.stop - cols.start, gen=gen)
    return x


def iterate(x):
    a, b, c = NS_COEFFICIENTS
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / x.norm().clamp_min(1e-7)
    for _ in range(5):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if tall else x


@pytest.mark.parametrize("kind", [gaussian, gradient, orthogonal, blocks])
@pytest.mark.parametrize("shape", SHAPES)
def test_error_beside_torch(shape, kind):
    x = kind(*shape, torch.Generator().manual_seed(sum(shape))).cuda()
    want = iterate(x.double())

    def error(y):
        return float((y.double() - want).norm() / want.norm())

    allowed = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        theirs = error(iterate(x))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = allowed
    assert error(newton_schulz(x)) < 1.5 * theirs + 1e-6
    assert native.device_error() == 0


@pytest.mark.parametrize("shape", [(40, 56), (100, 700), (150, 210), (300, 130)])
def test_non_finite_values_spread_over_the_matrix(shape):
    """One NaN or infinity on or off the gram's diagonal is a matrix of NaN, and no other's."""
    x = draw(*shape, gen=torch.Generator().manual_seed(1)).cuda()
    stack = torch.stack([x] * 4)
    stack[1, 0, 0], stack[2, 3, 7] = float("nan"), float("inf")
    got = newton_schulz(stack)
    assert torch.isnan(got[1]).all() and torch.isnan(got[2]).all()
    assert torch.equal(got[0], newton_schulz(x)) and torch.equal(got[3], got[0])


def test_coefficients_without_a_square():
    """c = 0 leaves A's own factor: the diagonal that is kept apart is not divided by it."""
    for shape in ((40, 56), (150, 210)):
        x = draw(*shape, gen=torch.Generator().manual_seed(2)).cuda()
        got = newton_schulz(x, steps=3, coefficients=(1.5, -0.5, 0.0)).double()
        y = x.double() / x.double().norm()
        for _ in range(3):
            y = 1.5 * y - 0.5 * y @ y.t() @ y
        assert float((got - y).norm() / y.norm()) < 1e-5
