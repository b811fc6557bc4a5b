"""
Forward-mode derivatives of the half-precision layer and of newton_schulz are
refused: neither has them, and a kernel that reads a dual tensor's memory would
return its value with the tangent lost.
"""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from create_graph_b200 import dense, native
from create_graph_b200 import library  # noqa: F401  (registers the operators)
from create_graph_b200.errors import NativeError
from create_graph_b200.optim import newton_schulz

ops = torch.ops.cg_b200
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def tensors(device):
    gen = torch.Generator().manual_seed(0)
    shapes = {"x": (6, 16), "weight": (8, 16), "bias": (8,), "residual": (6, 8)}
    return {name: torch.randn(*s, generator=gen).to(torch.bfloat16).to(device) for name, s in shapes.items()}


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["x", "weight", "bias", "residual"])
def test_linear(name, device):
    with forward_ad.dual_level():
        t = tensors(device)
        t[name] = dual(t[name])
        for call in (
            lambda: dense.linear(t["x"], t["weight"], t["bias"], residual=t["residual"]),
            lambda: ops.dense_linear(t["x"], t["weight"], t["bias"], t["residual"], "silu"),
        ):
            with pytest.raises(NativeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NativeError, match="forward-mode"):
                call()


@pytest.mark.parametrize("device", DEVICES)
def test_newton_schulz_and_gradient_operators(device):
    with forward_ad.dual_level():
        m = torch.randn(6, 8, device=device)
        h = m.to(torch.bfloat16)
        b = h[0].clone()
        calls = [lambda: newton_schulz(dual(m)), lambda: ops.newton_schulz(dual(m))]
        for i in range(2):
            args = [h, h.clone()]
            args[i] = dual(args[i])
            calls.append(lambda a=args: ops.act_grad(*a, "silu"))
        for i in range(4):
            args = [h, b, h.clone(), h.clone()]
            args[i] = dual(args[i])
            calls.append(lambda a=args: ops.act_grad2(*a, "silu"))
        for call in calls:
            with pytest.raises(NativeError, match="forward-mode"):
                call()


def test_tangent_of_the_incoming_gradient(monkeypatch):
    """Forward over reverse: the first-order backward would lose gy's tangent."""
    for name in ("_workspace_bytes", "_backward_workspace_bytes", "_stream"):
        monkeypatch.setattr(dense, name, lambda *a: 0)
    monkeypatch.setattr(native, "invoke", lambda *a, **k: None)
    t = tensors("cpu")
    x, w = t["x"].requires_grad_(True), t["weight"].requires_grad_(True)
    y = dense._Linear.apply(x, w, None, None, dense.ACTIVATIONS["silu"])[0]
    with forward_ad.dual_level():
        with pytest.raises(NativeError, match="forward-mode"):
            torch.autograd.grad(y, (x, w), dual(torch.ones(6, 8, dtype=torch.bfloat16)))


@pytest.mark.gpu
def test_plain_tensors_inside_a_dual_level():
    t = tensors("cuda")
    m = torch.randn(6, 8, device="cuda")
    want = dense.linear(t["x"], t["weight"], t["bias"], activation="gelu"), newton_schulz(m)
    with forward_ad.dual_level():
        got = dense.linear(t["x"], t["weight"], t["bias"], activation="gelu"), newton_schulz(m)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises((NativeError, RuntimeError)):
        torch.func.jvp(newton_schulz, (m,), (m,))
