"""
What the torch.library operators of the half-precision layer refuse before any
pointer reaches the library: tensors of another shape, type or device, and
layouts that the kernels would misread. The library is not called: a stand-in
records the arguments, and tensors on the CPU stand for ones on the GPU where a
call is expected to pass.
"""

from __future__ import annotations

import pytest
import torch

from create_graph_b200 import dense, native
from create_graph_b200 import library  # noqa: F401  (registers the operators)
from create_graph_b200.errors import NativeError

ops = torch.ops.cg_b200
BF16 = torch.bfloat16


class Scratch:
    @staticmethod
    def cg_act_grad_half_scratch_bytes(rows, cols):
        return 0


@pytest.fixture
def calls(monkeypatch):
    """The argument structs or arguments of the library calls that passed the checks."""
    seen = []

    def record(name, *args, info=None):
        seen.append((name, *(type(a._obj).from_buffer_copy(a._obj) if hasattr(a, "_obj") else a for a in args)))

    monkeypatch.setattr(native, "invoke", record)
    monkeypatch.setattr(native, "lib", lambda: Scratch)
    monkeypatch.setattr(native, "require_cuda", lambda *ts: None)
    monkeypatch.setattr(dense, "_stream", lambda t: 0)
    return seen


def matrix(rows, cols, dtype=BF16):
    return torch.randn(rows, cols).to(dtype)


def test_cpu_tensors_are_refused():
    gy = matrix(4, 8)
    with pytest.raises(NativeError, match="CUDA"):
        ops.act_grad(gy, gy.clone(), "silu")
    with pytest.raises(NativeError, match="CUDA"):
        ops.act_grad2(gy, gy[0].clone(), gy.clone(), gy.clone(), "silu")
    with pytest.raises(NativeError, match="CUDA"):
        ops.dense_linear(gy, gy.clone(), None, None, "silu")


GY = matrix(6, 8)


@pytest.mark.parametrize("z", [matrix(5, 8), matrix(6, 7), matrix(6, 8, torch.float16), matrix(6, 8, torch.float32),
                               torch.zeros(48, dtype=BF16)])
@pytest.mark.parametrize("activation", ["none", "silu"])
def test_act_grad_refuses_another_pre_activation(calls, z, activation):
    with pytest.raises(NativeError, match="act_grad: z is"):
        ops.act_grad(GY, z, activation)
    assert not calls


@pytest.mark.parametrize("name,bad", [(n, t) for n in ("h", "gy", "z") for t in
                                      (matrix(5, 8), matrix(6, 9), matrix(6, 8, torch.float16))]
                         + [("hb", torch.zeros(7, dtype=BF16)), ("hb", torch.zeros(8)), ("hb", matrix(1, 8))])
def test_act_grad2_refuses_unlike_tensors(calls, name, bad):
    given = {"h": GY, "hb": torch.zeros(8, dtype=BF16), "gy": matrix(6, 8), "z": matrix(6, 8), name: bad}
    with pytest.raises(NativeError, match="act_grad2"):
        ops.act_grad2(given["h"], given["hb"], given["gy"], given["z"], "gelu")
    assert not calls


def test_types_ranks_and_activations(calls):
    f32, cube = matrix(6, 8, torch.float32), torch.zeros(2, 3, 8, dtype=BF16)
    for call in (
        lambda: ops.act_grad(f32, f32.clone(), "silu"),
        lambda: ops.act_grad(cube, cube.clone(), "silu"),
        lambda: ops.act_grad(GY, GY.clone(), "tanh"),
        lambda: ops.act_grad2(f32, f32[0].clone(), f32.clone(), f32.clone(), "silu"),
        lambda: ops.act_grad2(GY, GY[0].clone(), GY.clone(), GY.clone(), "tanh"),
        lambda: ops.dense_linear(cube, GY, None, None, "none"),
    ):
        with pytest.raises(NativeError):
            call()
    assert not calls


def test_operands_of_a_gradient_product(calls):
    for b in (matrix(5, 7), matrix(5, 8, torch.float16), torch.zeros(5, 8, dtype=BF16, device="meta")):
        with pytest.raises(NativeError, match="gradient product"):
            dense._Product.apply(GY, b)
    assert not calls


def test_any_layout_of_the_pre_activation_is_read_by_rows(calls):
    z = matrix(8, 6).t()
    assert z.shape == (6, 8) and z.stride() == (1, 6)
    ops.act_grad(GY, z, "silu")
    (_, args, _), = calls
    assert args.z != z.data_ptr() and args.ld_z == 8 and (args.rows, args.cols) == (6, 8)
    wide = matrix(6, 20)[:, 2:10]
    ops.act_grad(GY, wide, "silu")
    assert calls[1][1].z == wide.data_ptr() and calls[1][1].ld_z == 20


def test_launches_on_the_tensors_own_device(monkeypatch):
    """Every launch happens with the device of the tensors current: the default
    stream has the same handle on all of them."""
    current, launched = [], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *exc):
            current.pop()

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(native, "invoke", lambda name, *a, **k: launched.append((name, tuple(current))))
    monkeypatch.setattr(native, "lib", lambda: Scratch)
    monkeypatch.setattr(native, "require_cuda", lambda *ts: None)
    monkeypatch.setattr(dense, "_stream", lambda t: 0)
    monkeypatch.setattr(dense, "_workspace_bytes", lambda *a: 0)
    ops.act_grad(GY, GY.clone(), "silu")
    ops.act_grad2(GY, GY[0].clone(), GY.clone(), GY.clone(), "silu")
    ops.dense_linear(GY, GY.clone(), None, None, "silu")
    index = GY.get_device()  # -1: the host's, which stands for the GPU's here
    assert launched == [(name, (index,)) for name in ("cg_act_grad_half", "cg_act_grad2_half", "cg_linear_half")]


@pytest.mark.gpu
def test_layouts_on_the_gpu():
    gen = torch.Generator().manual_seed(3)
    gy, z = (torch.randn(70, 40, generator=gen).to(torch.float16).cuda() for _ in range(2))
    h, hb = torch.randn(70, 40, generator=gen).to(torch.float16).cuda(), gy[0].clone()
    want, want2 = ops.act_grad(gy, z, "gelu"), ops.act_grad2(h, hb, gy, z, "gelu")
    turned = z.t().contiguous().t()
    wide = torch.zeros(70, 64, dtype=torch.float16, device="cuda")[:, 5:45].copy_(z)
    for other in (turned, wide):
        got, got2 = ops.act_grad(gy, other, "gelu"), ops.act_grad2(h, hb, gy, other, "gelu")
        assert torch.equal(got[0], want[0]) and torch.equal(got2[0], want2[0]) and torch.equal(got2[1], want2[1])
        # the chunks of the column sums follow the layout: a few fp32 roundings, then one of fp16
        assert float((got[1].double() - want[1].double()).norm()) <= 2.0**-10 * float(want[1].double().norm())
    with pytest.raises(NativeError, match="z is"):
        ops.act_grad(gy, z[:8], "gelu")
    with pytest.raises(NativeError, match="z is"):
        ops.act_grad(gy, z.cpu(), "gelu")
    with pytest.raises(NativeError, match="hb is"):
        ops.act_grad2(h, hb[:8], gy, z, "gelu")
