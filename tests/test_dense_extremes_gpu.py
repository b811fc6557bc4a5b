"""
The half-precision dense layer's activations at the ends of their range: NaN,
infinities and values far from zero, on each of its ways of storing a result
(aligned rows, odd pitches, k split over several tiles, both kinds of them).

Layers are built so that a chosen value is the pre-activation itself: x holds it
in one column, weight has a one there, so z is exact in fp32.
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


def one_per_row(values, n, k, dtype):
    """x (len(values), k) and weight (n, k) with z[i, j] = values[i] for even j, 0 for odd j."""
    x = torch.zeros(len(values), k, dtype=dtype)
    x[:, 1] = torch.tensor(values, dtype=torch.float64).to(dtype)
    w = torch.zeros(n, k, dtype=dtype)
    w[::2, 1] = 1.0
    return x.cuda(), w.cuda()


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
