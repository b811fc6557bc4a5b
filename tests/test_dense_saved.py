"""
What the half-precision dense layer's backward reads when a saved-tensor hook
gives the saved tensors back in another layout: the pitch and major order that
reach the library have to be those of the tensor whose address goes with them.

The library is not called: a stand-in records the arguments of each call and
the tensors live on the CPU. The values are compared on a GPU.
"""

from __future__ import annotations

import pytest
import torch

from create_graph_b200 import dense, native
from create_graph_b200.errors import NativeError


@pytest.fixture
def calls(monkeypatch):
    """(name, arguments) of the library calls made, the argument structs copied."""
    seen = []

    def record(name, *args, info=None):
        seen.append((name, *(type(a._obj).from_buffer_copy(a._obj) if hasattr(a, "_obj") else a for a in args)))

    monkeypatch.setattr(native, "invoke", record)
    monkeypatch.setattr(dense, "_stream", lambda t: 0)
    monkeypatch.setattr(dense, "_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(dense, "_backward_workspace_bytes", lambda *a: 0)
    return seen


def backward_call(calls, x, w, pack, unpack, act="silu"):
    """The backward's argument struct and the tensors that the hook gave back."""
    back = []

    def unpacked(t):
        back.append(unpack(t))
        return back[-1]

    with torch.autograd.graph.saved_tensors_hooks(pack, unpacked):
        y = dense._Linear.apply(x, w, None, None, dense.ACTIVATIONS[act])[0]
    torch.autograd.grad(y, (x, w), torch.ones_like(y))
    (args,) = [c[1] for c in calls if c[0] == "cg_linear_half_backward"]
    return args, back


def reads(address, pitch, mn_major, t):
    """Whether (address, pitch, major order) is the tensor t as it lies in memory."""
    rows, cols = (1, 0) if mn_major else (0, 1)
    return address == t.data_ptr() and (t.stride(cols) == 1 or t.shape[cols] == 1) and \
        (pitch == t.stride(rows) or t.shape[rows] == 1)


def aligned(*shape):
    t = torch.randn(*shape).to(torch.bfloat16)
    assert t.data_ptr() % 16 == 0
    return t


PACKS = {
    "clone to rows": lambda t: t.clone(memory_format=torch.contiguous_format),
    "clone to columns": lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone(),
    "wider rows": lambda t: torch.empty(t.shape[0], 2 * t.shape[1] + 8, dtype=t.dtype, device=t.device)[:, : t.shape[1]].copy_(t)
    if t.dim() == 2 else t.clone(),
}


@pytest.mark.parametrize("pack", sorted(PACKS))
@pytest.mark.parametrize("form", ["rows", "slice", "transposed"])
def test_backward_reads_saved_tensors_as_they_come_back(calls, form, pack):
    m, n, k = 32, 24, 16
    make = {"rows": aligned, "slice": lambda r, c: aligned(r, 200)[:, :c], "transposed": lambda r, c: aligned(c, r).t()}
    x, w = (make[form](*s).detach().requires_grad_(True) for s in ((m, k), (n, k)))
    args, back = backward_call(calls, x, w, PACKS[pack], lambda t: t)
    x1, w1, z1 = [t for t in back if t.dim() == 2]
    assert reads(args.x, args.ld_x, args.x_mn_major, x1)
    assert reads(args.w, args.ld_w, args.w_mn_major, w1)
    assert args.ld_z >= n
    if z1.stride(1) == 1:
        assert reads(args.z, args.ld_z, False, z1)
    else:  # copied to rows
        assert args.z != z1.data_ptr() and args.ld_z == n


def test_saved_rows_off_the_boundary_are_copied(calls):
    m, n, k = 32, 24, 16
    x, w = (aligned(*s).requires_grad_(True) for s in ((m, k), (n, k)))

    def off(t):  # rows three values off a 16-byte boundary
        return torch.empty(t.shape[0], t.shape[1] + 5, dtype=t.dtype)[:, 3 : 3 + t.shape[1]].copy_(t)

    args, back = backward_call(calls, x, w, off, lambda t: t, act="none")
    (pad,) = [c[1:] for c in calls if c[0] == "cg_pad_rows_half"]
    x1, w1 = back
    # (source, its pitch, rows, columns, copy, its pitch) twice
    assert pad[:4] == (x1.data_ptr(), k + 5, m, k) and pad[6:10] == (w1.data_ptr(), k + 5, n, k)
    assert (args.x, args.ld_x) == pad[4:6] and (args.w, args.ld_w) == pad[10:12]


def test_padded_copies_follow_their_buffer(calls):
    """Operands that the forward copied are read from the buffer as it comes back."""
    x, w = (aligned(*s).requires_grad_(True) for s in ((32, 13), (24, 13)))
    args, back = backward_call(calls, x, w, lambda t: t.clone(), lambda t: t)
    (flat,) = [t for t in back if t.dim() == 1]
    assert args.x == flat.data_ptr() and args.ld_x == args.ld_w == 16
    assert args.w == flat.data_ptr() + 2 * 32 * 16


def test_recorded_backward_reads_the_pre_activation_by_rows(calls):
    x, w = (aligned(*s).requires_grad_(True) for s in ((32, 16), (24, 16)))
    back = []
    with torch.autograd.graph.saved_tensors_hooks(PACKS["clone to columns"], lambda t: back.append(t) or t):
        y = dense._Linear.apply(x, w, None, None, dense.ACTIVATIONS["gelu"])[0]
    torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    (args,) = [c[1] for c in calls if c[0] == "cg_act_grad_half"]
    (z,) = [t for t in back if t.shape == (32, 24)]
    assert z.stride() == (1, 32) and args.z != z.data_ptr() and args.ld_z == 24


@pytest.mark.parametrize("pack", [lambda t: t.float(), lambda t: t[:-1]])
def test_other_saved_tensors_are_refused(calls, pack):
    x, w = (aligned(*s).requires_grad_(True) for s in ((32, 16), (24, 16)))
    with pytest.raises(NativeError, match="saved tensor"):
        backward_call(calls, x, w, pack, lambda t: t)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("form", ["rows", "slice", "transposed", "odd"])
def test_gradients_under_hooks(form, act):
    """The gradients do not depend on the layout the saved tensors come back in:
    the products' order of summation does not follow it."""
    m, n, k = 130, 96, 72
    gen = torch.Generator().manual_seed(1)
    draw = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).cuda()  # noqa: E731
    make = {"rows": draw, "slice": lambda r, c: draw(r, 2304)[:, 8 : 8 + c], "transposed": lambda r, c: draw(c, r).t(),
            "odd": lambda r, c: draw(r, c + 1)[:, 1:]}
    x, w = (make[form](*s).detach().requires_grad_(True) for s in ((m, k), (n, k)))
    gy = draw(m, n)

    def grads():
        return torch.autograd.grad(dense.linear(x, w, activation=act), (x, w), gy)

    want = grads()
    hooks = [torch.autograd.graph.save_on_cpu(pin_memory=pin) for pin in (False, True)]
    hooks += [torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t) for pack in PACKS.values()]
    for hook in hooks:
        with hook:
            y = dense.linear(x, w, activation=act)
        got = torch.autograd.grad(y, (x, w), gy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert native.device_error() == 0
