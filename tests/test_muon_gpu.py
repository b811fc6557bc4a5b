"""
Newton-Schulz orthogonalisation (optim.newton_schulz) and the Muon step
(optim.FusedMuon) against the definitions in float64, and their refusals.

Tolerances, norm-wise relative. The iteration runs on pairs of fp16 planes (22
significant bits) with fp32 accumulation: one product is off by about 2^-22
sqrt(3) and its accumulation by 2^-24 per 16-deep step, and an error in a weak
direction grows by a = 3.4445 per step while that direction does the same, so
relative to the result five steps of three products stay near 15 x 2^-22 =
4e-6 for matrices of full rank: 1e-5 in fp32. A low-rank matrix feeds the
rounding of its strong directions (2^-22) into the empty ones, which grow by
3.4445^5 = 485: 485 x 2^-22 = 1.2e-4. Half-precision outputs add one rounding
(2^-8 or 2^-11).
"""

from __future__ import annotations

import pytest
import torch

from create_graph_b200 import native
from create_graph_b200.ddp import FlatGradients
from create_graph_b200.errors import NativeError
from create_graph_b200.optim import NS_COEFFICIENTS, FusedAdamW, FusedMuon, newton_schulz

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 1e-5, torch.float16: 2.0**-11 + 1e-5, torch.bfloat16: 2.0**-8 + 1e-5}
LOW_RANK = 485 * 2.0**-22


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


def orthogonalised(x, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = x.detach().double()
    x = x / x.norm(dim=(-2, -1), keepdim=True).clamp_min(eps)
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            g = x @ x.mT
            x = a * x + (b * g + c * g @ g) @ x
        else:
            g = x.mT @ x
            x = a * x + x @ (b * g + c * g @ g)
    return x


def random(*shape, dtype=torch.float32, seed=0, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (9, 1), (8, 8), (33, 65), (65, 33), (128, 128), (127, 129),
                                   (3, 130, 257), (2, 257, 130), (4, 64, 200), (300, 700), (1031, 260), (2, 3, 40, 24),
                                   (640, 640), (17, 3000), (100, 1024), (1024, 100), (128, 512), (385, 128),
                                   (7, 129, 64), (128, 1025), (40, 16, 16)])
def test_against_definition(shape, dtype):
    x = random(*shape, dtype=dtype, seed=1)
    got = newton_schulz(x)
    assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous()
    assert rel(got, orthogonalised(x)) < TOL[dtype]
    assert native.device_error() == 0


@pytest.mark.parametrize("shape", [(768, 768), (2304, 768), (768, 3072), (3072, 768)])
def test_model_shapes(shape):
    strong = random(shape[0], 32, seed=2) @ random(32, shape[1], seed=3)
    x = 1e-4 * (strong / 32**0.5 + random(*shape, seed=4))
    got = newton_schulz(x)
    assert rel(got, orthogonalised(x)) < TOL[torch.float32]
    s = torch.linalg.svdvals(got.double())
    assert float(s.max()) < 1.3
    if shape[0] != shape[1]:  # the smallest singular values of a square random matrix are near zero
        assert 0.3 < float(s.min())


@pytest.mark.parametrize("shape", [(96, 160), (260, 256)])
def test_low_rank(shape):
    x = random(shape[0], 8, seed=5) @ random(8, shape[1], seed=6)
    assert rel(newton_schulz(x), orthogonalised(x)) < LOW_RANK


def test_extreme_scales_zero_and_non_finite():
    x = random(40, 56, seed=7)
    want = newton_schulz(x)
    for scale in (2.0**-80, 2.0**80):  # powers of two: nothing is rounded
        assert torch.equal(newton_schulz(x * scale, eps=1e-38), want)
    tiny = newton_schulz(x * 2.0**-40)  # below eps: divided by eps instead
    assert rel(tiny, orthogonalised(x * 2.0**-40)) < TOL[torch.float32]
    stack = torch.stack([x, torch.zeros_like(x), x])
    stack[2, 3, 5] = float("nan")
    got = newton_schulz(stack)
    assert torch.equal(got[0], want) and not got[1].any() and torch.isnan(got[2]).all()


def test_steps_and_coefficients():
    x = random(70, 50, seed=8)
    for steps, coefficients in ((1, NS_COEFFICIENTS), (2, NS_COEFFICIENTS), (12, (1.5, -0.5, 0.0)), (3, (2.0, -1.5, 0.5))):
        got = newton_schulz(x, steps=steps, coefficients=coefficients)
        # at most 3 products a step
        assert rel(got, orthogonalised(x, steps, coefficients)) < max(1e-5, 3 * steps * 2.0**-22)


def test_strides_batches_streams_and_repeats():
    x = random(5, 48, 72, seed=9)
    want = newton_schulz(x)
    assert torch.equal(newton_schulz(x[3]), want[3])
    wide = torch.zeros(5, 50, 99, device="cuda")
    wide[:, :48, :72] = x
    assert torch.equal(newton_schulz(wide[:, :48, :72]), want)
    wide[:, 1:49, 3:75] = x
    assert torch.equal(newton_schulz(wide[:, 1:49, 3:75]), want)
    assert torch.equal(newton_schulz(x.mT.contiguous().mT), want)
    assert torch.equal(newton_schulz(x[::2]), want[::2])
    assert torch.equal(newton_schulz(x[:1].expand(3, 48, 72)), want[:1].expand(3, 48, 72))
    assert rel(newton_schulz(x.mT), want.mT) < TOL[torch.float32]
    assert newton_schulz(x[:0]).shape == (0, 48, 72) and newton_schulz(x[:, :0]).shape == (5, 0, 72)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = newton_schulz(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want)


def muon_reference(w, g, m, lr, mu, wd, nesterov):
    m = m + (1 - mu) * (g - m)
    u = g + mu * (m - g) if nesterov else m
    rate = lr * max(1.0, w.shape[0] / w.shape[1]) ** 0.5
    return (1 - lr * wd) * w - rate * orthogonalised(u), m


# more shapes than one launch takes, repeated ones, odd ones, single rows
SHAPES = [(37, 11), (64, 128), (128, 64), (37, 11), (1, 9), (130, 130), (12, 100), (100, 12), (64, 128), (5, 5),
          (48, 16), (16, 48), (64, 128)]


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps(nesterov):
    gen = torch.Generator().manual_seed(10)
    init = [torch.randn(*s, generator=gen) for s in SHAPES]
    params = [torch.nn.Parameter(t.clone().cuda()) for t in init]
    grads = FlatGradients(params, None)
    opt = FusedMuon(grads, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.2)
    assert all(p.data_ptr() >= opt.flat.data_ptr() for p in params)
    ref = [(t.double(), torch.zeros_like(t, dtype=torch.float64)) for t in init]
    for step in range(3):
        if step == 2:
            opt.lr = 0.01
        gs = [torch.randn(*s, generator=gen) for s in SHAPES]
        grads.zero()
        for p, g in zip(params, gs):
            p.grad.copy_(g)
        opt.step()
        ref = [muon_reference(w, g.double(), m, opt.lr, 0.9, 0.2, nesterov) for (w, m), g in zip(ref, gs)]
        for p, (w, _), (o, n), (_, m) in zip(params, ref, grads.offsets, ref):
            assert rel(p, w) < 3 * TOL[torch.float32]
            assert rel(opt.momentum_buffer[o : o + n].view_as(p), m) < 1e-6
    assert native.device_error() == 0
    # the gaps between the slices stay zero
    inside = torch.zeros_like(opt.flat, dtype=torch.bool)
    for o, n in grads.offsets:
        inside[o : o + n] = True
    assert not opt.flat[~inside].any() and not opt.momentum_buffer[~inside].any()


@pytest.mark.parametrize("shapes", [[(24, 40), (40, 24)] * 40, [(160, 140), (140, 160)] * 16,
                                    [(16, 20), (300, 30), (30, 700), (150, 136), (1000, 90)] * 12])
def test_muon_many_matrices_in_one_step(shapes):
    # more runs than one launch's table takes, more clusters than the SMs hold at once
    gen = torch.Generator().manual_seed(11)
    params = [torch.nn.Parameter(torch.randn(*s, generator=gen).cuda()) for s in shapes]
    before = [p.detach().double().cpu() for p in params]
    grads = FlatGradients(params, None)
    opt = FusedMuon(grads, lr=0.1, weight_decay=0.0)
    gs = [torch.randn(*s, generator=gen) for s in shapes]
    for p, g in zip(params, gs):
        p.grad.copy_(g)
    opt.step()
    for p, w, g in zip(params, before, gs):
        want, _ = muon_reference(w, g.double(), torch.zeros_like(w), 0.1, 0.95, 0.0, True)
        assert rel(p, want) < 3 * TOL[torch.float32]


def test_muon_captured_graph_and_full_decay():
    p = torch.nn.Parameter(random(64, 96, seed=12))
    grads = FlatGradients([p], None)
    p.grad.copy_(random(64, 96, seed=13))
    opt = FusedMuon(grads, lr=0.5, weight_decay=2.0, momentum=0.0)  # 1 - lr wd = 0: the old weights vanish
    opt.step()
    want, _ = muon_reference(torch.zeros(64, 96).double(), p.grad.double().cpu(), torch.zeros(64, 96).double(), 0.5,
                             0.0, 0.0, True)
    assert rel(p, want) < TOL[torch.float32]
    first = p.detach().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    p.data.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), first)


def test_beside_adamw():
    """Matrices with Muon, the rest with AdamW: a regression both learn."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(12, 32), torch.nn.SiLU(), torch.nn.Linear(32, 3)).cuda()
    matrices = [p for p in model.parameters() if p.dim() == 2]
    rest = [p for p in model.parameters() if p.dim() != 2]
    flat = [FlatGradients(matrices, None), FlatGradients(rest, None)]
    opts = [FusedMuon(flat[0], lr=0.02), FusedAdamW(flat[1], lr=0.01)]
    x = random(256, 12, seed=14)
    y = torch.stack([x[:, 0] * x[:, 1], x[:, 2].sin(), x[:, 3]], 1)
    losses = []
    for _ in range(150):
        for f in flat:
            f.zero()
        loss = (model(x) - y).square().mean()
        loss.backward()
        for o in opts:
            o.step()
        losses.append(float(loss))
    assert losses[-1] < 0.3 * losses[0]


def test_refusals():
    x = random(8, 6)
    for call in (
        lambda: newton_schulz(x.double()),
        lambda: newton_schulz(x[0]),
        lambda: newton_schulz(x.cpu()),
        lambda: newton_schulz(x, steps=0),
        lambda: newton_schulz(x, eps=0.0),
        lambda: newton_schulz(x, coefficients=(1.0, 2.0)),
        lambda: newton_schulz(x, coefficients=(1.0, 2.0, float("nan"))),
        lambda: newton_schulz(x.clone().requires_grad_(True)),
    ):
        with pytest.raises(NativeError):
            call()
    with torch.no_grad():
        newton_schulz(x.clone().requires_grad_(True))
    vector = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError, match="matrices"):
        FusedMuon(FlatGradients([vector], None))
    matrix = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    with pytest.raises(ValueError, match="momentum"):
        FusedMuon(FlatGradients([matrix], None), momentum=1.0)
    with pytest.raises(ValueError, match="float32"):
        FusedMuon(FlatGradients([torch.nn.Parameter(torch.zeros(4, 4, device="cuda").half())], None))
    args = native.NsArgs()
    entry = native.NsEntry()
    large = random(200, 160)  # smaller matrices need no workspace
    entry.x = entry.out = large.data_ptr()
    entry.rows, entry.cols, entry.count, entry.ld_x, entry.ld_out = 200, 160, 1, 160, 160
    args.entries, args.n, args.steps, args.eps = native.ctypes.pointer(entry), 1, 5, 1e-7
    with pytest.raises(NativeError, match="workspace"):
        native.invoke("cg_newton_schulz", args, 0)
    entry.ld_x = 159
    with pytest.raises(NativeError, match="pitch"):
        native.invoke("cg_newton_schulz", args, 0)
