"""
The half-precision dense layer (create_graph_b200.dense) against the formula in
float64, its first and second derivatives, and its refusals.

Tolerances, norm-wise relative, u = 2^-8 (bf16) or 2^-11 (fp16) the unit
roundoff: an output rounded once is off by at most u; a gradient that passes
through one more rounded value (gz) and the kept pre-activation by at most 3 u
(each rounding at most u, f'' z / f' below 1 on average); a second-order term
passes through four to five roundings, 8 u. fp32 accumulation adds less than
2^-11 sqrt(K) 2^-11.
"""

from __future__ import annotations

import pytest
import torch

from create_graph_b200 import native
from create_graph_b200.dense import ACTIVATIONS, Linear, linear
from create_graph_b200.errors import NativeError

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
DTYPES = [torch.bfloat16, torch.float16]


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


def formula(x, w, b, r, act):
    z = x @ w.t()
    if b is not None:
        z = z + b
    f = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}
    y = f[act](z)
    return y if r is None else y + r


def tensors(m, n, k, dtype, bias=True, residual=True, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def draw(*s, scale=1.0):
        return (scale * torch.randn(*s, generator=gen)).to(dtype).cuda()

    return (draw(m, k), draw(n, k, scale=k**-0.5 if k else 1.0), draw(n) if bias else None,
            draw(m, n) if residual else None, draw(m, n))


def doubled(*ts):
    return [None if t is None else t.detach().double().cpu().requires_grad_(True) for t in ts]


SIZES = [(1, 8, 8), (1, 1000, 768), (2, 3, 5), (7, 64, 1), (128, 64, 64), (129, 257, 65), (300, 200, 100),
         (1000, 2304, 768), (77, 3072, 768), (5, 4096, 40), (4099, 1031, 515), (1, 1, 20000), (256, 256, 8192)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mnk", SIZES)
def test_forward_sizes(mnk, dtype):
    x, w, b, r, _ = tensors(*mnk, dtype)
    for act, bias, res in (("none", None, None), ("silu", b, r), ("gelu", b, None), ("relu", None, r)):
        got = linear(x, w, bias, activation=act, residual=res)
        want = formula(*doubled(x, w, bias, res), act)
        assert got.shape == want.shape and got.dtype == dtype and got.is_contiguous()
        assert rel(got, want.detach()) < 1.1 * UNIT[dtype], (mnk, act)
    assert native.device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
@pytest.mark.parametrize("mnk", [(64, 128, 512), (130, 96, 264), (33, 17, 9), (1, 24, 40), (2100, 768, 256)])
def test_gradients(mnk, act, dtype):
    x, w, b, r, gy = tensors(*mnk, dtype, seed=1)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = linear(x, w, b, activation=act, residual=r)
    got = torch.autograd.grad(y, leaves, gy)
    ref = doubled(x, w, b, r)
    want = torch.autograd.grad(formula(*ref, act), ref, gy.double().cpu())
    for name, g, e in zip(("dx", "dw", "db", "dr"), got, want):
        assert g.shape == e.shape and g.dtype == dtype
        assert rel(g, e) < 3.0 * UNIT[dtype], (name, rel(g, e))
    assert torch.equal(got[3], gy)
    assert native.device_error() == 0


@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
@pytest.mark.parametrize("mnk", [(2, 1, 19), (35, 1, 8), (300, 1, 264), (1, 1, 1), (70, 2, 1), (1, 37, 50)])
def test_gradients_of_thin_layers(mnk, act):
    """One or two columns, one row: incoming gradients whose layout says little.
    A gradient may be a single sum of signed terms here, so the error is held
    against the sum of their magnitudes: 3 u |gy| (|f'| + |z f''| <= 1.5)."""
    dtype = torch.bfloat16
    x, w, b, _, gy = tensors(*mnk, dtype, seed=13)
    wide = torch.zeros(mnk[0], mnk[1] + 7, dtype=dtype, device="cuda")
    column = wide[:, 3 : 3 + mnk[1]]
    column.copy_(gy)
    ref = doubled(x, w, b)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    # the last one: a gradient of ones with no memory of its own
    for g in (gy, column, gy.t().contiguous().t(), torch.ones((), dtype=dtype, device="cuda").expand(mnk[:2])):
        got = torch.autograd.grad(linear(x, w, b, activation=act), leaves, g)
        gd = g.double().cpu()
        want = torch.autograd.grad(formula(*ref, None, act), ref, gd)
        size = 1.5 * gd.abs()
        sizes = (size @ ref[1].detach().abs(), size.t() @ ref[0].detach().abs(), size.sum(0))
        for a, e, s in zip(got, want, sizes):
            assert float((a.double().cpu() - e).norm()) < 3.0 * UNIT[dtype] * float(s.norm())


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_against_differences(act):
    # directional derivative of <gy, y> along a random direction of x, central
    # differences of the float64 formula with step 2^-10 (error of order step^2
    # = 1e-6, below the layer's 3 u)
    x, w, b, r, gy = tensors(65, 72, 48, torch.float16, seed=2)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(linear(x, w, b, activation=act, residual=r), x, gy)
    d = torch.randn(65, 48, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    xd, wd, bd, rd = (t.detach() for t in doubled(x, w, b, r))
    g, h = gy.double().cpu(), 2.0**-10
    up, down = (formula(xd + s * h * d, wd, bd, rd, act) for s in (1, -1))
    want = float((g * (up - down)).sum() / (2 * h))
    got = float((dx.double().cpu() * d).sum())
    scale = float(dx.double().cpu().norm() * d.norm())
    assert abs(got - want) < 3.0 * UNIT[torch.float16] * scale


@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
@pytest.mark.parametrize("mnk", [(40, 24, 16), (129, 67, 35)])
def test_second_order(mnk, act):
    """The parameter gradient through an input gradient, as force training takes it."""
    dtype = torch.float16
    x, w, b, r, gy = tensors(*mnk, dtype, seed=4)
    v = torch.randn(mnk[0], mnk[2], generator=torch.Generator().manual_seed(5)).to(dtype).cuda()

    def run(f, x, w, b, gy, v):
        y = f(x, w, b)
        (dx,) = torch.autograd.grad(y, x, gy, create_graph=True)
        return torch.autograd.grad((dx * v).sum(), (w, gy) if act in ("none", "relu") else (x, w, b, gy),
                                   allow_unused=True)

    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, gy)]
    got = run(lambda x, w, b: linear(x, w, b, activation=act), *leaves, v)
    ref = doubled(x, w, b, gy)
    want = run(lambda x, w, b: formula(x, w, b, None, act), *ref, v.double().cpu())
    for i, (g, e) in enumerate(zip(got, want)):
        assert rel(g, e) < 8.0 * UNIT[dtype], (i, rel(g, e))


def test_second_order_through_bias_gradient():
    dtype = torch.float16
    x, w, b, _, gy = tensors(50, 40, 24, dtype, seed=6)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    hb = torch.randn(40, generator=torch.Generator().manual_seed(7)).to(dtype).cuda()
    (db,) = torch.autograd.grad(linear(x, w, b, activation="silu"), b, gy, create_graph=True)
    got = torch.autograd.grad((db * hb).sum(), leaves)
    ref = doubled(x, w, b)
    (db,) = torch.autograd.grad(formula(*ref, None, "silu"), ref[2], gy.double().cpu(), create_graph=True)
    want = torch.autograd.grad((db * hb.double().cpu()).sum(), ref)
    for g, e in zip(got, want):
        assert rel(g, e) < 8.0 * UNIT[dtype]


def test_views_and_leading_dimensions():
    dtype = torch.bfloat16
    x, w, b, r, _ = tensors(96, 80, 64, dtype, seed=8)
    want = formula(*(t.detach() for t in doubled(x, w, b, r)), "silu")
    tol = 1.1 * UNIT[dtype]
    wide = torch.zeros(96, 200, dtype=dtype, device="cuda")
    cases = []
    for offset in (0, 8, 3):  # aligned, aligned at an offset, unaligned
        wide[:, offset : offset + 64] = x
        cases.append(linear(wide[:, offset : offset + 64].clone(memory_format=torch.preserve_format), w, b,
                            activation="silu", residual=r))
        view = torch.empty_like(wide)[:, offset : offset + 64]
        view.copy_(x)
        cases.append(linear(view, w, b, activation="silu", residual=r))
    cases.append(linear(x.t().contiguous().t(), w.t().contiguous().t(), b, activation="silu", residual=r))
    res = torch.empty(96, 83, dtype=dtype, device="cuda")[:, 1:81]
    res.copy_(r)
    cases.append(linear(x, w, b, activation="silu", residual=res))
    cases.append(linear(x, w, b, activation="silu", residual=r.t().contiguous().t()))
    cases.append(linear(x.view(4, 24, 64), w, b, activation="silu", residual=r.view(4, 24, 80)).view(96, 80))
    cases.append(torch.stack([linear(x[i], w, b, activation="silu", residual=r[i]) for i in (0, 95)]))
    for got in cases[:-1]:
        assert rel(got, want) < tol
    assert rel(cases[-1], want[[0, 95]]) < tol
    # one row repeated by a zero stride
    got = linear(x[:1].expand(96, 64), w, b)
    assert torch.equal(got, linear(x[:1], w, b).expand(96, 80))


@pytest.mark.parametrize("mnk", [(0, 24, 16), (5, 0, 16), (5, 24, 0)])
def test_empty(mnk):
    x, w, b, r, gy = tensors(*mnk, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = linear(x, w, b, activation="silu", residual=r)
    ref = doubled(x, w, b, r)
    want = formula(*ref, "silu")
    assert y.shape == want.shape
    if y.numel():
        assert rel(y, want.detach()) < 1.1 * UNIT[torch.bfloat16]
    for g, e in zip(torch.autograd.grad(y, leaves, gy), torch.autograd.grad(want, ref, gy.double().cpu())):
        assert g.shape == e.shape and rel(g, e) < 3.0 * UNIT[torch.bfloat16]


def test_non_finite_values_stay_in_their_rows():
    x, w, b, r, _ = tensors(300, 128, 64, torch.bfloat16, seed=9)
    clean = linear(x, w, b, activation="none", residual=r)
    x = x.clone()
    x[17, 3], x[250, 0] = float("inf"), float("nan")
    got = linear(x, w, b, activation="none", residual=r)
    rows = torch.ones(300, dtype=torch.bool)
    rows[[17, 250]] = False
    assert torch.equal(got[rows.cuda()], clean[rows.cuda()])
    assert not torch.isfinite(got[17]).any() and torch.isnan(got[250]).all()
    big = torch.full((4, 8), 300.0, dtype=torch.float16, device="cuda")
    assert torch.isinf(linear(big, big)).all()  # 8 * 9e4 overflows fp16, as it does when rounded


def test_same_result_every_run_and_on_another_stream():
    x, w, b, r, gy = tensors(700, 264, 4096, torch.bfloat16, seed=10)  # split over k
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]

    def step():
        y = linear(x, w, b, activation="gelu", residual=r)
        return (y, *torch.autograd.grad(y, leaves, gy))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


def test_module_and_captured_graph():
    torch.manual_seed(0)
    layer = Linear(64, 48, activation="silu").cuda()
    x = torch.randn(32, 64, dtype=torch.bfloat16, device="cuda")
    want = layer(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), torch.no_grad():
        layer(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = layer(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_refusals():
    x, w, b, r, _ = tensors(16, 24, 8, torch.bfloat16)
    for call in (
        lambda: linear(x.float(), w.float()),
        lambda: linear(x, w.half()),
        lambda: linear(x, w[:, :4]),
        lambda: linear(x, w, b[:5]),
        lambda: linear(x, w, b.float()),
        lambda: linear(x, w, b, residual=r[:3]),
        lambda: linear(x, w, b, activation="tanh"),
        lambda: linear(x.cpu(), w, b),
        lambda: linear(x, w.cpu(), b),
        lambda: linear(x, w[0]),
    ):
        with pytest.raises(NativeError):
            call()
    args = native.LinearArgs()
    args.m = args.n = args.k = 8
    args.lda = args.ldb = args.ld_y = 8
    args.a, args.b, args.y, args.dtype = x.data_ptr(), w.data_ptr(), x.data_ptr(), native.F32
    with pytest.raises(NativeError, match="dtype"):
        native.invoke("cg_linear_half", args, 0)
    args.dtype, args.lda = native.BF16, 9
    with pytest.raises(NativeError, match="multiples of 8"):
        native.invoke("cg_linear_half", args, 0)
    args.lda, args.a = 8, x.data_ptr() + 2
    with pytest.raises(NativeError, match="aligned"):
        native.invoke("cg_linear_half", args, 0)


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_library_operators(act):
    """torch.ops.cg_b200.dense_linear, differentiated twice, and newton_schulz."""
    import create_graph_b200.library  # noqa: F401
    from create_graph_b200.optim import newton_schulz

    dtype = torch.float16
    x, w, b, r, gy = tensors(72, 40, 24, dtype, seed=11)
    v = torch.randn(72, 24, generator=torch.Generator().manual_seed(12)).to(dtype).cuda()

    def run(f, x, w, b, r, gy, v):
        y = f(x, w, b, r)
        dx, dw, db, dr = torch.autograd.grad(y, (x, w, b, r), gy, create_graph=True)
        second = torch.autograd.grad((dx * v).sum(), (w, gy), allow_unused=True)
        return y, dx, dw, db, dr, *second

    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r, gy)]
    got = run(lambda x, w, b, r: torch.ops.cg_b200.dense_linear(x, w, b, r, act)[0], *leaves, v)
    ref = doubled(x, w, b, r, gy)
    want = run(lambda *t: formula(*t, act), *ref, v.double().cpu())
    for i, (g, e) in enumerate(zip(got, want)):
        assert rel(g.detach(), e.detach()) < (1.1 if i == 0 else 3.0 if i < 5 else 8.0) * UNIT[dtype], i
    m = torch.randn(30, 20, device="cuda")
    assert torch.equal(torch.ops.cg_b200.newton_schulz(m), newton_schulz(m))
