"""
The half-precision dense layer and the matrix optimizer without a GPU: refusals
on the host, the shapes of their torch.library operators, and a traced double
backward. Tensors on a GPU are covered by test_dense_gpu.py and test_muon_gpu.py.
"""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import create_graph_b200.library  # noqa: F401  (registers the operators)
from create_graph_b200.ddp import FlatGradients
from create_graph_b200.dense import Linear, linear
from create_graph_b200.errors import NativeError
from create_graph_b200.optim import FusedMuon, newton_schulz

ops = torch.ops.cg_b200


def test_no_cpu_fallback():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(NativeError, match="CUDA"):
        linear(x, w)
    with pytest.raises(NativeError, match="CUDA"):
        newton_schulz(torch.zeros(4, 4))
    with pytest.raises(NativeError, match="CUDA"):
        Linear(8, 6)(x)
    grads = FlatGradients([torch.nn.Parameter(torch.zeros(4, 6))], None)
    with pytest.raises(NativeError, match="CUDA"):
        FusedMuon(grads).step()


def test_refusals_before_any_launch():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(NativeError, match="activation"):
        linear(x, w, activation="tanh")
    with pytest.raises(NativeError, match="float16 or bfloat16"):
        linear(x.float(), w.float())
    with pytest.raises(NativeError, match="activation"):
        Linear(8, 6, activation="tanh")
    with pytest.raises(NativeError, match="float16 or bfloat16"):
        Linear(8, 6, dtype=torch.float32)
    for bad in (torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(2, 3, 4))):
        with pytest.raises(ValueError, match="matrices"):
            FusedMuon(FlatGradients([bad], None))
    matrix = [torch.nn.Parameter(torch.zeros(3, 4))]
    with pytest.raises(ValueError, match="momentum"):
        FusedMuon(FlatGradients(matrix, None), momentum=-0.1)
    with pytest.raises(NativeError, match="steps"):
        FusedMuon(FlatGradients(matrix, None), steps=0)


def test_muon_keeps_parameters_in_its_flat_buffer():
    params = [torch.nn.Parameter(torch.randn(5, 7)), torch.nn.Parameter(torch.randn(16, 4))]
    before = [p.detach().clone() for p in params]
    opt = FusedMuon(FlatGradients(params, None))
    assert all(torch.equal(p, b) for p, b in zip(params, before))
    for p, (offset, n) in zip(params, opt.grads.offsets):
        assert p.data_ptr() == opt.flat.data_ptr() + 4 * offset and offset % 64 == 0 and n == p.numel()
    assert not opt.momentum_buffer.any()


def test_module_keeps_float32_parameters():
    layer = Linear(8, 6, activation="silu")
    assert layer.weight.dtype == layer.bias.dtype == torch.float32 and layer.weight.shape == (6, 8)
    assert Linear(8, 6, bias=False).bias is None


def test_fake_shapes():
    with FakeTensorMode():
        dev, bf16 = "cuda", torch.bfloat16
        x, w = torch.empty(40, 16, device=dev, dtype=bf16), torch.empty(24, 16, device=dev, dtype=bf16)
        b, r = torch.empty(24, device=dev, dtype=bf16), torch.empty(40, 24, device=dev, dtype=bf16)
        y, z = ops.dense_linear(x, w, b, r, "silu")
        assert y.shape == z.shape == (40, 24) and y.dtype == bf16
        gz, db = ops.act_grad(y, z, "silu")
        assert gz.shape == y.shape and db.shape == (24,)
        dgy, dz = ops.act_grad2(gz, db, y, z, "silu")
        assert dgy.shape == dz.shape == y.shape
        m = torch.empty(3, 20, 50, device=dev)
        assert ops.newton_schulz(m).shape == m.shape


def test_traced_double_backward():
    def force_loss(x, w, b):
        y, _ = ops.dense_linear(x, w, b, None, "silu")
        e = ops.dense_linear(y, w.t().contiguous(), None, y.new_zeros(y.shape[0], w.shape[1]), "gelu")[0].sum()
        (g,) = torch.autograd.grad(e, x, create_graph=True)
        return torch.autograd.grad(g.float().square().sum(), (w, b))

    # fake CPU tensors: the autograd engine would look for a CUDA context for
    # fake CUDA ones, and the fakes do not depend on the device
    with FakeTensorMode():
        bf16 = torch.bfloat16
        x = torch.empty(12, 16, dtype=bf16, requires_grad=True)
        w = torch.empty(24, 16, dtype=bf16, requires_grad=True)
        b = torch.empty(24, dtype=bf16, requires_grad=True)
        graph = make_fx(force_loss, tracing_mode="fake")(x, w, b)
    called = {str(node.target) for node in graph.graph.nodes}
    for name in ("dense_linear", "act_grad", "act_grad2"):
        assert f"cg_b200.{name}.default" in called, called
