"""
The half-precision dense layer's activations at the ends of their range: NaN,
infinities and values far from zero, on each of its ways of storing a result
(aligned rows, odd pitches, k split over several tiles, both kinds of them).

Chosen pre-activations come through the bias of a layer whose weight is zero, so
they are exact. At the infinities the activations and their derivatives take
their limits.
"""

from __future__ import annotations

import pytest
import torch

from create_graph_b200 import native
from create_graph_b200.dense import linear

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
DTYPES = sorted(UNIT, key=str)
ACTS = ["none", "relu", "silu", "gelu"]
NAN, INF = float("nan"), float("inf")
# outputs n and inner length k: aligned rows, odd pitches, and few tiles of a
# long k (split) with either
FORMS = [(64, 64), (37, 40), (64, 8192), (37, 8192)]


def far_values(dtype):
    """Values of the type from its ends to where the activations bend."""
    big = float(torch.finfo(dtype).max)
    mid = [1e4, 300.0, 100.0, 64.0, 43.5, 41.0, 20.0, 9.0, 3.0]
    values = [INF, big, *([1e30, 1e20] if dtype == torch.bfloat16 else [3e4]), *mid, 0.5]
    return torch.tensor([*values, 0.0, *(-v for v in values)], dtype=torch.float64).to(dtype).double()


def by_bias(n, k, dtype):
    """(x, weight, bias, z): a layer of three rows whose pre-activations are its bias."""
    z = far_values(dtype)[torch.arange(n) % len(far_values(dtype))]
    x = torch.randn(3, k, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    return x, torch.zeros(n, k, dtype=dtype, device="cuda"), z.to(dtype).cuda(), z.expand(3, n)


def limit(f, z, low):
    """f(z) in float64, ``low`` at -infinity and z at infinity."""
    y = f(z)
    return torch.where(z == -INF, torch.full_like(z, low), torch.where(z == INF, z, y))


FORMULA = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
           "gelu": lambda z: 0.5 * z * torch.special.erfc(-z * 0.5**0.5)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n,k", FORMS)
def test_nan_stays_nan_and_in_its_place(n, k, act, dtype):
    """A NaN in the bias is a column of NaN, one in the residual an element, one
    in x a row; every other value is as without it."""
    gen = torch.Generator().manual_seed(1)
    x, w, b, r = (torch.randn(*s, generator=gen).to(dtype).cuda() for s in ((33, k), (n, k), (n,), (33, n)))
    clean = linear(x, w, b, activation=act, residual=r)
    b2, r2, x2 = b.clone(), r.clone(), x.clone()
    b2[6], r2[4, 9], x2[20, 3] = NAN, NAN, NAN
    got = linear(x2, w, b2, activation=act, residual=r2)
    bad = torch.zeros(33, n, dtype=torch.bool, device="cuda")
    bad[:, 6] = bad[4, 9] = bad[20] = True
    assert torch.isnan(got[bad]).all()
    assert torch.equal(got[~bad], clean[~bad])
    assert native.device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n,k", FORMS)
def test_values_far_from_zero(n, k, act, dtype):
    """One rounding, and 1e-16 beside it: silu is held at 9e-18 below -43, gelu's
    tail is right to a hundredth where it is 5e-15. fp16 rounds to steps of 2^-24
    near zero."""
    x, w, b, z = by_bias(n, k, dtype)
    got = linear(x, w, b, activation=act).double().cpu()
    want = limit(FORMULA[act], z, -INF if act == "none" else 0.0)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    step = 2.0**-25 if dtype == torch.float16 else 0.0
    error = (got - want)[~inf].abs()
    assert (error <= 1.1 * UNIT[dtype] * want[~inf].abs() + 1e-16 + step).all(), float(error.max())
