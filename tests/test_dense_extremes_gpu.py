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

from create_graph_b200 import library  # noqa: F401  (registers the operators)
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


def derivative(act, z):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        d = torch.sigmoid(z) * (1.0 + z * torch.sigmoid(-z))
    else:
        d = 0.5 * torch.special.erfc(-z * 0.5**0.5) + z * torch.exp(-0.5 * z * z) / (2.0 * torch.pi) ** 0.5
    return torch.where(torch.isinf(z), (z > 0).double(), d)


def bias_gradient(x, w, b, act, recorded):
    """f'(z) itself: the bias gradient of a layer with one row and an incoming gradient of ones."""
    b = b.detach().requires_grad_(True)
    w = w.detach().requires_grad_(True)
    y = linear(x, w, b, activation=act)
    dw, db = torch.autograd.grad(y, (w, b), torch.ones_like(y), create_graph=recorded)
    return dw.detach(), db.detach().double().cpu()


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n,k", FORMS[:2])
def test_derivative_far_from_zero(n, k, act, dtype, recorded):
    """One rounding, and beside it 43 ulps of 1 (silu: 1 - s times z, 5.2e-6; Phi is
    right to 1.5e-7) and fp16's steps of 2^-24 near zero."""
    x, w, b, z = by_bias(n, k, dtype)
    dw, got = bias_gradient(x[:1], w, b, act, recorded)
    want = derivative(act, z[0])
    step = 2.0**-25 if dtype == torch.float16 else 0.0
    error = (got - want).abs()
    assert (error <= 1.1 * UNIT[dtype] * want.abs() + 5.2e-6 + step).all(), z[0][error.argmax()]
    assert torch.isfinite(dw).all()


@pytest.mark.parametrize("act,low,high", [("relu", 0.0, 1.0), ("silu", 0.0, 1.0), ("gelu", 0.0, 1.0)])
@pytest.mark.parametrize("n", [64, 37])
def test_derivative_where_the_kept_value_left_its_type(n, act, low, high):
    """z = +-90000 is beyond fp16: the output is 0 or infinity, the gradient 0 or 1."""
    for sign, want in ((-1.0, low), (1.0, high)):
        x = torch.full((1, 1), 300.0, dtype=torch.float16, device="cuda")
        w = torch.full((n, 1), 300.0 * sign, dtype=torch.float16, device="cuda")
        b = torch.zeros(n, dtype=torch.float16, device="cuda")
        y = linear(x, w, b, activation=act)
        assert (y == 0).all() if sign < 0 else torch.isinf(y).all()
        assert (bias_gradient(x, w, b, act, False)[1] == want).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("n", [64, 37])
def test_derivative_of_nan(n, act):
    x, w, b, _ = by_bias(n, 40, torch.bfloat16)
    clean = bias_gradient(x[:1], w, b, act, False)[1]
    b[6] = NAN
    got = bias_gradient(x[:1], w, b, act, False)[1]
    assert torch.isnan(got[6])
    got[6] = clean[6]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_second_derivative_far_from_zero(act, dtype):
    """f'' is 0 at both ends; bounds as for f'."""
    z = torch.cat([far_values(dtype), torch.tensor([NAN], dtype=torch.float64)])
    if act == "silu":
        s = torch.sigmoid(z)
        want = s * torch.sigmoid(-z) * (2.0 + z * (torch.sigmoid(-z) - s))
    elif act == "gelu":
        want = torch.exp(-0.5 * z * z) * (2.0 - z * z) / (2.0 * torch.pi) ** 0.5
    else:
        want = torch.zeros_like(z)
    want = torch.where(z.abs() > 1e4, torch.zeros_like(z), want)  # below 1e-1000
    one = torch.ones(1, z.numel(), dtype=dtype, device="cuda")
    none = torch.zeros(z.numel(), dtype=dtype, device="cuda")
    got = torch.ops.cg_b200.act_grad2(one, none, one.clone(), z.to(dtype).cuda()[None], act)[1].double().cpu()[0]
    if act in ("silu", "gelu"):
        assert torch.isnan(got[-1])
    step = 2.0**-25 if dtype == torch.float16 else 0.0
    error = (got - want)[:-1].abs()
    assert (error <= 1.1 * UNIT[dtype] * want[:-1].abs() + 5.2e-6 + step).all(), z[error.argmax()]
