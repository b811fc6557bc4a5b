"""
The half-precision dense layer: y = f(x W^T + b) + r in one product.

    y = dense.linear(x, weight, bias, activation="silu", residual=r)

bf16 or fp16 tensors, fp32 accumulation on the tcgen05 tensor cores, bias,
activation and residual applied to the fp32 accumulator and rounded once
(``cg_linear_half``). ``activation`` is "none", "relu", "silu" or "gelu" (the
erf form). x is (..., K), weight (N, K), bias (N,), residual (..., N); all have
one dtype. Transposed and row-strided views of x and weight are read in place
when their rows start on 16-byte boundaries; others are copied once.

The op is differentiable twice, as the force pass of ``cg.create_graph`` needs:

    gz = gy f'(z);  dx = gz W;  dW = gz^T x;  db = sum of gz;  dr = gy

with gz and db formed in one pass over gy and the kept pre-activation z, the
gradients as products of the same kernel, and the second order (f'') as an
explicit kernel. gz is rounded to the layer's dtype before the two products,
as every operand of the tensor cores is. Without a gradient to prepare, z is
not written. NaN stays NaN; at infinite pre-activations, also ones beyond the
type's range, f, f' and f'' take their limits. Third and forward-mode
derivatives are refused. The fp32 layers of the energy network are in
``create_graph_b200.nn``.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch import Tensor, nn

from create_graph_b200 import native
from create_graph_b200.compile_config import engine_will_execute
from create_graph_b200.errors import NativeError
from create_graph_b200.nn import _edges, _Fused

ACTIVATIONS = {"none": native.ACT_NONE, "relu": native.ACT_RELU, "silu": native.ACT_SILU, "gelu": native.ACT_GELU}


def _pitched(rows: int, cols: int, like: Tensor) -> Tensor:
    """An uninitialised (rows, cols) matrix whose rows start on 16-byte boundaries."""
    pitch = -(-cols // 8) * 8
    out = torch.empty(rows, pitch, dtype=like.dtype, device=like.device)
    return out if pitch == cols else out[:, :cols]


def _fits_tma(t: Tensor, row: int, col: int) -> bool:
    """Whether t, contiguous along dimension ``col``, can be read in place by
    TMA: 16-byte aligned base and row pitch, rows that do not overlap."""
    pitch = t.stride(row) if t.shape[row] > 1 else -(-t.shape[col] // 8) * 8
    return (t.stride(col) == 1 or t.shape[col] == 1) and pitch % 8 == 0 and pitch >= t.shape[col] \
        and t.data_ptr() % 16 == 0


def _matrix_like(t: Tensor, like: Tensor) -> Tensor:
    """An uninitialised contiguous matrix of t's shape."""
    return torch.empty_like(t) if t.is_contiguous() else like.new_empty(t.shape)


def _stream(t: Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _in_place(t: Tensor):
    """(None, row pitch, MN-major) of a logical (rows, K) operand that the
    products can read as it is stored; None when its rows need copying."""
    if t.is_contiguous():  # the usual case, in few steps
        k = t.shape[1]
        if k % 8 == 0 and t.data_ptr() % 16 == 0:
            return None, k, False
    if _fits_tma(t, 0, 1):
        return None, t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8, False
    if _fits_tma(t, 1, 0):
        return None, t.stride(1) if t.shape[1] > 1 else -(-t.shape[0] // 8) * 8, True
    return None


def _operands(*ts: Tensor) -> tuple[list, Tensor | None]:
    """How the products read one or two operands, as (offset, row pitch,
    MN-major) each, and a buffer: an offset of None is the tensor itself, else
    the place (in values) of its copy in the buffer, with padded rows and in the
    operand's own layout (a transposed view stays transposed). One launch copies
    them all."""
    ops = [_in_place(t) for t in ts]
    if None not in ops:
        return ops, None
    todo, at = [], 0
    for i, t in enumerate(ts):
        if ops[i] is None:
            mn = t.stride(0) == 1 and t.stride(1) >= t.shape[0]
            stored = t.t() if mn else _rows(t)
            pitch = -(-stored.shape[1] // 8) * 8
            ops[i] = (at, pitch, mn)
            todo.append((stored, at, pitch))
            at += stored.shape[0] * pitch
    flat = ts[0].new_empty(at)
    args = []
    for stored, at, pitch in todo:
        rows, cols = stored.shape
        args += [stored.data_ptr(), max(stored.stride(0), cols), rows, cols, flat.data_ptr() + 2 * at, pitch]
    native.invoke("cg_pad_rows_half", *args, *([None, 0, 0, 0, None, 0] if len(todo) == 1 else []), _stream(ts[0]))
    return ops, flat


def _saved_operands(ops, strides, flat: Tensor | None, x: Tensor, w: Tensor) -> tuple[list, Tensor | None]:
    """The forward's operands as a backward may read them from the saved tensors:
    a copy where the forward left it in the buffer; a tensor that was read in
    place as then, or asked for its layout again where a saved-tensor hook
    (save_on_cpu, or any pack that clones) gave it back in another one."""
    if flat is not None:
        if not flat.is_contiguous() or flat.data_ptr() % 16 != 0:
            return _operands(x, w)
    elif x.data_ptr() % 16 == 0 and w.data_ptr() % 16 == 0 and (x.stride(), w.stride()) == strides:
        return ops, None  # the usual case
    ops = [_in_place(t) if op[0] is None else op for op, t in zip(ops, (x, w))]
    return _operands(x, w) if None in ops else (ops, flat)


def _require(what: str, t: Tensor, shape: tuple[int, ...], like: Tensor) -> None:
    """Refuse a tensor that the kernels would misread (its strides may be any)."""
    if t.shape != shape or t.dtype is not like.dtype or t.device != like.device:
        raise NativeError(f"{what} is {tuple(t.shape)} {t.dtype} on {t.device}, expected {tuple(shape)} {like.dtype} "
                          f"on {like.device}")


def _address(t: Tensor, op, flat: Tensor | None) -> int:
    return t.data_ptr() if op[0] is None else flat.data_ptr() + 2 * op[0]


def _rows(t: Tensor) -> Tensor:
    """t with unit column stride (a copy when it has none)."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(m: int, n: int, k: int) -> int:
    args = native.LinearArgs()
    args.m, args.n, args.k = m, n, k
    return native.lib().cg_linear_half_workspace_bytes(ctypes.byref(args))


@functools.lru_cache(maxsize=4096)
def _backward_workspace_bytes(m: int, n: int, k: int, act: int, dx: bool, dw: bool, db: bool) -> int:
    args = native.LinearBackwardArgs()
    args.m, args.n, args.k, args.act = m, n, k, act
    args.dx, args.dw, args.db = 16 * dx or None, 16 * dw or None, 16 * db or None  # only whether they are wanted
    return native.lib().cg_linear_half_backward_workspace_bytes(ctypes.byref(args))


def _forward(a, b, ops, flat, shape, bias, activation, residual, keep_z):
    """(y, z) of one product of operands a and b as _operands gives them."""
    m, n, k = shape
    y = a.new_empty((m, n))
    z = torch.empty_like(y) if keep_z else None
    args = native.LinearArgs()
    args.m, args.n, args.k = m, n, k
    (_, args.lda, args.a_mn_major), (_, args.ldb, args.b_mn_major) = ops
    args.a, args.b = _address(a, ops[0], flat), _address(b, ops[1], flat)
    if bias is not None:
        bias = bias.contiguous()
        args.bias = bias.data_ptr()
    if residual is not None:
        residual = _rows(residual)
        args.residual, args.ld_residual = residual.data_ptr(), max(residual.stride(0), n)
    if z is not None:
        args.z, args.ld_z = z.data_ptr(), n
    args.y, args.ld_y = y.data_ptr(), n
    args.act, args.dtype = activation, native.HALF_DTYPES[a.dtype]
    nbytes = _workspace_bytes(m, n, k)
    workspace = None
    if nbytes > 0:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=a.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), nbytes
    native.invoke("cg_linear_half", ctypes.byref(args), _stream(a), info=(m, n, k))
    return y, z


def product(a: Tensor, b: Tensor, bias: Tensor | None = None, activation: int = native.ACT_NONE,
            residual: Tensor | None = None, keep_z: bool = False):
    """(y, z) with z = a @ b.T + bias and y = f(z) + residual; z is None unless
    ``keep_z``. a (M, K), b (N, K), either of them possibly a transposed view."""
    m, k = a.shape
    n = b.shape[0]
    if m == 0 or n == 0:
        y = torch.empty(m, n, dtype=a.dtype, device=a.device)
        return y, torch.empty_like(y) if keep_z else None
    if k == 0:  # an empty sum: zero columns give it
        a, b, k = a.new_zeros(m, 8), b.new_zeros(n, 8), 8
    return _forward(a, b, *_operands(a, b), (m, n, k), bias, activation, residual, keep_z)


def _backward(gy, z, x, w, ops, flat, shape, activation, want_dx, want_dw, want_db):
    """(dx, dw, db) in one call; None for what is not wanted."""
    m, n, k = shape
    pitch = -(-n // 8) * 8
    args = native.LinearBackwardArgs()
    args.m, args.n, args.k, args.act, args.dtype = m, n, k, activation, native.HALF_DTYPES[gy.dtype]
    gz = None
    if activation == native.ACT_NONE:
        if _fits_tma(gy, 0, 1):
            args.gy, args.ld_gy = gy.data_ptr(), gy.stride(0) if m > 1 else pitch
        else:
            # rows on 16-byte boundaries, whatever other layout would do
            gy = gy.contiguous()
            kept = gy.new_empty(m * pitch)
            args.gy, args.ld_gy = kept.data_ptr(), pitch
            native.invoke("cg_pad_rows_half", gy.data_ptr(), n, m, n, args.gy, pitch, None, 0, 0, 0, None, 0,
                          _stream(gy))
    else:
        if not gy.is_contiguous():
            gy = _rows(gy)
        if not z.is_contiguous():
            z = _rows(z)
        gz = torch.empty_like(z) if pitch == n and z.is_contiguous() else gy.new_empty((m, pitch))
        args.gy, args.ld_gy = gy.data_ptr(), max(gy.stride()[0], n)
        args.z, args.ld_z = z.data_ptr(), max(z.stride()[0], n)
        args.gz, args.ld_gz = gz.data_ptr(), pitch
    (_, args.ld_x, args.x_mn_major), (_, args.ld_w, args.w_mn_major) = ops
    args.x, args.w = _address(x, ops[0], flat), _address(w, ops[1], flat)
    dx = _matrix_like(x, gy) if want_dx else None
    dw = _matrix_like(w, gy) if want_dw else None
    db = gy.new_empty(n) if want_db else None
    args.dx, args.dw, args.db = native.ptr(dx), native.ptr(dw), native.ptr(db)
    nbytes = _backward_workspace_bytes(m, n, k, activation, want_dx, want_dw, want_db)
    workspace = None
    if nbytes > 0:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=gy.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), nbytes
    native.invoke("cg_linear_half_backward", ctypes.byref(args), _stream(gy), info=(m, n, k))
    return dx, dw, db


def _act_grad(gy: Tensor, z: Tensor | None, activation: int, want_db: bool):
    """(gz, db): gz = gy f'(z) (gy itself without an activation), db its column
    sums or None."""
    if z is not None:
        _require("dense.act_grad: z", z, gy.shape, gy)
    gy = _rows(gy)
    rows, cols = gy.shape
    args = native.ActGradArgs()
    args.rows, args.cols, args.act, args.dtype = rows, cols, activation, native.HALF_DTYPES[gy.dtype]
    args.gy, args.ld_gy = gy.data_ptr(), max(gy.stride(0), cols)
    gz, db, scratch = gy, None, None
    if activation != native.ACT_NONE:
        z = _rows(z)
        gz = _pitched(rows, cols, gy)
        args.z, args.ld_z = z.data_ptr(), max(z.stride(0), cols)
        args.gz, args.ld_gz = gz.data_ptr(), max(gz.stride(0), cols)
    if want_db:
        db = torch.empty(cols, dtype=gy.dtype, device=gy.device)
        nbytes = native.lib().cg_act_grad_half_scratch_bytes(rows, cols)
        scratch = torch.empty(max(nbytes // 4, 1), dtype=torch.float32, device=gy.device)
        args.db, args.scratch, args.scratch_bytes = db.data_ptr(), scratch.data_ptr(), nbytes
    if args.gz or args.db:
        native.invoke("cg_act_grad_half", ctypes.byref(args), _stream(gy))
    return gz, db


class _Product(_Fused):
    """C = a @ b.T; backward: g @ b and g.T @ a."""

    @staticmethod
    def forward(ctx, a, b):
        _require("dense.linear: operand of a gradient product", b, (b.shape[0], a.shape[1]), a)
        ctx.save_for_backward(a, b)
        ctx.edges = _edges(a, b)
        return product(a, b)[0]

    @staticmethod
    def backward(ctx, g):
        a, b = ctx.saved_tensors
        ga = _Product.apply(g, b.t()) if ctx.needs_input_grad[0] and engine_will_execute(ctx.edges[0]) else None
        gb = _Product.apply(g.t(), a.t()) if ctx.needs_input_grad[1] and engine_will_execute(ctx.edges[1]) else None
        return ga, gb


class _ActGrad(_Fused):
    """(gz, db) of _act_grad; backward: the second-order kernel."""

    @staticmethod
    def forward(ctx, gy, z, activation, want_db):
        ctx.save_for_backward(gy, z)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        gz, db = _act_grad(gy, z, activation, want_db)
        return (gz.view_as(gz) if gz is gy else gz), db

    @staticmethod
    def backward(ctx, h, hb):
        gy, z = ctx.saved_tensors
        if h is None and hb is None:
            return None, None, None, None
        if z is None:  # no activation: gz is gy
            t = hb.expand(gy.shape) if h is None else h if hb is None else h + hb
            return t, None, None, None
        return *_ActGrad2.apply(h, hb, gy, z, ctx.activation), None, None


def _act_grad2(h: Tensor | None, hb: Tensor | None, gy: Tensor, z: Tensor, activation: int):
    """((h + hb) f'(z), (h + hb) gy f''(z)); either cotangent may be None."""
    _require("dense.act_grad2: z", z, gy.shape, gy)
    if h is not None:
        _require("dense.act_grad2: h", h, gy.shape, gy)
    if hb is not None:
        _require("dense.act_grad2: hb", hb, gy.shape[1:], gy)
    h = None if h is None else h.contiguous()
    hb = None if hb is None else hb.contiguous()
    gy, z = gy.contiguous(), z.contiguous()
    dgy, dz = torch.empty_like(gy), torch.empty_like(z)
    native.invoke("cg_act_grad2_half", native.ptr(h), native.ptr(hb), gy.data_ptr(), z.data_ptr(), dgy.data_ptr(),
                  dz.data_ptr(), gy.shape[0], gy.shape[1], activation, native.HALF_DTYPES[gy.dtype], _stream(gy))
    return dgy, dz


class _ActGrad2(_Fused):
    """_act_grad2: the last derivative the force training needs."""

    @staticmethod
    def forward(ctx, h, hb, gy, z, activation):
        return _act_grad2(h, hb, gy, z, activation)

    @staticmethod
    def backward(ctx, *grads):
        raise NativeError("dense.linear: third derivatives are not supported")


# below this many flops a product takes less time (15 us) than finding out which
# results were asked for (8 us per input, on the host)
_SMALL_FLOPS = 2e10


class _Linear(_Fused):
    """(y, z) from one product; z is None without an activation."""

    @staticmethod
    def forward(ctx, x, w, b, r, activation):
        ctx.activation = activation
        ctx.shape = m, n, k = x.shape[0], w.shape[0], x.shape[1]
        # z is seldom used: its gradient arrives as None, not as zeros
        ctx.set_materialize_grads(False)
        keep_z = activation != native.ACT_NONE
        ctx.operands = flat = None
        if min(m, n, k) == 0:
            y, z = product(x, w, b, activation, r, keep_z)
        else:
            ctx.operands, flat = _operands(x, w)
            ctx.strides = x.stride(), w.stride()
            y, z = _forward(x, w, ctx.operands, flat, ctx.shape, b, activation, r, keep_z)
        ctx.save_for_backward(x, w, z, flat)
        ctx.inputs = (True, True, b is not None)
        return y, z

    @staticmethod
    def _wanted(ctx, need, recording):
        """Which of x, w, b the backward pass running now needs."""
        m, n, k = ctx.shape
        if 2.0 * m * n * k < _SMALL_FLOPS and not recording:
            return need
        nodes = iter(ctx.next_functions)
        nodes = [next(nodes)[0] if given else None for given in ctx.inputs]
        return [n and engine_will_execute(node) for n, node in zip(need, nodes)]

    @staticmethod
    def backward(ctx, gy, gz_direct):
        x, w, z, flat = ctx.saved_tensors
        native.refuse_tangents("dense.linear", gy, gz_direct, x, w, z)
        *need, need_dr, _ = ctx.needs_input_grad
        recording = torch.is_grad_enabled()
        want = _Linear._wanted(ctx, need, recording)
        dr = gy if need_dr else None
        if not recording and gz_direct is None and gy is not None and ctx.operands is not None:
            if not any(want):
                return None, None, None, dr, None
            m, n, k = ctx.shape
            like = gy.dtype, gy.get_device()
            if x.shape != (m, k) or w.shape != (n, k) or (x.dtype, x.get_device()) != like or \
                    (w.dtype, w.get_device()) != like:
                _require("dense.linear: saved tensor x", x, (m, k), gy)
                _require("dense.linear: saved tensor weight", w, (n, k), gy)
            if z is not None:
                _require("dense.linear: saved tensor z", z, (m, n), gy)
            ops, flat = _saved_operands(ctx.operands, ctx.strides, flat, x, w)
            return *_backward(gy, z, x, w, ops, flat, ctx.shape, ctx.activation, *want), dr, None
        # the differentiable path: products and passes that record their own backward
        gz, db = gz_direct, None
        if gy is not None and any(want):
            alone = gz_direct is None
            gz, db = _ActGrad.apply(gy, z, ctx.activation, want[2] and alone)
            if not alone:
                gz = gz + gz_direct
        if gz is None:
            return None, None, None, dr, None
        if want[2] and db is None:
            db = _ActGrad.apply(gz, None, native.ACT_NONE, True)[1]
        dx = _Product.apply(gz, w.t()) if want[0] else None
        dw = _Product.apply(gz.t(), x.t()) if want[1] else None
        return dx, dw, db, dr, None


def _activation(who: str, name: str) -> int:
    act = ACTIVATIONS.get(name)
    if act is None:
        raise NativeError(f"{who}: activation must be one of {sorted(ACTIVATIONS)}, got {name!r}")
    return act


def _checked_matrix(who: str, gy: Tensor, activation: str, *others: Tensor) -> int:
    """The activation's code; refuses a gy that is no half-precision matrix on
    the GPU, and tangents of it or the others."""
    act = _activation(who, activation)
    native.refuse_tangents(who, gy, *others)
    if gy.dim() != 2 or gy.dtype not in native.HALF_DTYPES:
        raise NativeError(f"{who}: a float16 or bfloat16 matrix expected, got {tuple(gy.shape)} {gy.dtype}")
    native.require_cuda(gy)
    return act


def _checked(x, weight, bias, residual, activation) -> int:
    act = _activation("dense.linear", activation)
    native.refuse_tangents("dense.linear", x, weight, bias, residual)
    dtype, device = x.dtype, x.device
    if dtype not in native.HALF_DTYPES:
        raise NativeError(f"dense.linear: float16 or bfloat16 expected, got {dtype} (the fp32 layers are in "
                          "create_graph_b200.nn)")
    native.require_cuda(x)
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and (t.dtype != dtype or t.device != device):
            raise NativeError(f"dense.linear: {name} is {t.dtype} on {t.device}, x {dtype} on {device}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise NativeError(f"dense.linear: x {tuple(x.shape)} does not match weight {tuple(weight.shape)}")
    n = weight.shape[0]
    if bias is not None and tuple(bias.shape) != (n,):
        raise NativeError(f"dense.linear: bias must be ({n},), got {tuple(bias.shape)}")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], n):
        raise NativeError(f"dense.linear: residual must be {(*x.shape[:-1], n)}, got {tuple(residual.shape)}")
    return act


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str = "none",
           residual: Tensor | None = None) -> Tensor:
    """f(x @ weight.T + bias) + residual (see the module's description)."""
    act = _checked(x, weight, bias, residual, activation)
    if x.get_device() != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return linear(x, weight, bias, activation=activation, residual=residual)
    shape = x.shape
    if x.dim() != 2:
        x = x.reshape(math.prod(shape[:-1]), shape[-1])
        residual = None if residual is None else residual.reshape(x.shape[0], weight.shape[0])
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        y = _Linear.apply(x, weight, bias, residual, act)[0]
    else:
        y = product(x, weight, bias, act, residual)[0]
    return y if len(shape) == 2 else y.view(*shape[:-1], weight.shape[0])


class Linear(nn.Module):
    """A half-precision layer y = f(x W^T + b) + r, initialised as
    torch.nn.Linear. The parameters are kept in float32, as the optimizers and
    ``ddp.FlatGradients`` want them, and rounded to ``dtype`` for each product;
    their gradients come back as float32."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "none",
                 dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        if dtype not in native.HALF_DTYPES:
            raise NativeError(f"dense.Linear: float16 or bfloat16 expected, got {dtype}")
        _activation("dense.Linear", activation)
        self.activation, self.dtype = activation, dtype
        like = nn.Linear(in_features, out_features, bias=bias, device=device, dtype=torch.float32)
        self.weight, self.bias = like.weight, like.bias

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Tensor:
        bias = None if self.bias is None else self.bias.to(self.dtype)
        return linear(x, self.weight.to(self.dtype), bias, activation=self.activation, residual=residual)
