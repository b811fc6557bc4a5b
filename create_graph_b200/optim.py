"""
The optimizer updates of the training step: AdamW and Muon over the flat
buffers, and the Newton-Schulz orthogonalisation that Muon is built on.

``FusedAdamW(flat_grads)`` moves the parameters of a ``ddp.FlatGradients``
into one flat fp32 buffer laid out like its gradient buffer (each parameter's
``.data`` becomes a view into it, on a 256-byte boundary like a separate
allocation, so weights keep their TMA-friendly alignment), keeps the two
moment buffers beside it,
and applies torch.optim.AdamW's update (amsgrad off) to all of them with one
kernel launch per step (``cg_adamw_step``). The reference ships no optimizer:
its training loops use torch's; this is the fused equivalent for the step
that follows ``loss.backward()`` and the gradient all-reduce.

``FusedMuon(flat_grads)`` does the same for the matrices of a model: momentum,
an orthogonalised update and weight decay in one call for all of them
(``cg_muon_step``). Give it a ``FlatGradients`` of the 2-D weights and
``FusedAdamW`` another one of everything else (embeddings, biases, norms):

    matrices = [p for name, p in model.named_parameters() if p.dim() == 2 and "embed" not in name]
    rest = [p for p in model.parameters() if all(p is not m for m in matrices)]
    muon = FusedMuon(FlatGradients(matrices, world), lr=1e-3)
    adamw = FusedAdamW(FlatGradients(rest, world), lr=1e-3)

``newton_schulz(x)`` is the orthogonalisation alone, for a matrix or a stack.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from create_graph_b200 import native
from create_graph_b200.ddp import FlatGradients
from create_graph_b200.errors import NativeError

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_NS_DTYPES = {torch.float32: native.F32, **native.HALF_DTYPES}


def _into_flat(grads: FlatGradients) -> Tensor:
    """The parameters moved into one buffer of the gradient buffer's layout
    (256-byte aligned slices, zero gaps that the updates keep at zero)."""
    flat = torch.zeros_like(grads.flat)
    with torch.no_grad():
        for p, (offset, n) in zip(grads.params, grads.offsets):
            view = flat[offset : offset + n].view_as(p)
            view.copy_(p)
            p.data = view
    return flat


class FusedAdamW:
    def __init__(self, grads: FlatGradients, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2):
        if grads.flat.dtype != torch.float32:
            raise ValueError("FusedAdamW: parameters must be float32")
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"FusedAdamW: betas {betas} outside [0, 1)")
        self.grads = grads
        self.flat = _into_flat(grads)
        self.exp_avg = torch.zeros_like(self.flat)
        self.exp_avg_sq = torch.zeros_like(self.flat)
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        # step count and bias corrections on the device (cg_adamw_step_counted),
        # so that a CUDA graph holding the update replays the next step each time
        self.state = torch.zeros(2, dtype=torch.int64, device=self.flat.device)

    @property
    def steps(self) -> int:
        """Steps taken so far (reads the device counter: synchronises)."""
        return int(self.state[0])

    @torch.no_grad()
    def step(self) -> None:
        native.call("cg_adamw_step_counted", self.flat.data_ptr(), self.grads.flat.data_ptr(),
                    self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), self.flat.numel(), self.lr, self.betas[0],
                    self.betas[1], self.eps, self.weight_decay, self.state.data_ptr(),
                    native.stream_ptr(self.flat.device))


def _ns_args(who: str, dtype: torch.dtype, steps: int, coefficients, eps: float) -> native.NsArgs:
    if dtype not in _NS_DTYPES:
        raise NativeError(f"{who}: float32, float16 or bfloat16 expected, got {dtype}")
    if steps < 1:
        raise NativeError(f"{who}: steps must be at least 1, got {steps}")
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise NativeError(f"{who}: three finite coefficients expected, got {coefficients!r}")
    if not (math.isfinite(eps) and eps > 0.0):
        raise NativeError(f"{who}: eps must be positive, got {eps}")
    args = native.NsArgs()
    args.dtype, args.steps, args.eps = _NS_DTYPES[dtype], steps, eps
    args.a, args.b, args.c = coefficients
    return args


def _ns_workspace(args: native.NsArgs, device: torch.device) -> Tensor:
    nbytes = native.lib().cg_newton_schulz_workspace_bytes(ctypes.byref(args))
    workspace = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = workspace.data_ptr(), nbytes
    return workspace


def newton_schulz(x: Tensor, steps: int = 5, coefficients: tuple[float, float, float] = NS_COEFFICIENTS,
                  eps: float = 1e-7) -> Tensor:
    """Each matrix of x (..., m, n) with its singular values s / |x| driven
    towards 1 by ``steps`` applications of a s + b s^3 + c s^5:

        X = x / max(|x|, eps);  X <- a X + (b A + c A A) X,  A = X X^T

    (from the right when m > n). float32, float16 or bfloat16 in and out; the
    iteration itself runs at fp32-level accuracy whatever the type, because it
    multiplies the error of the weak directions by a in every step. A matrix of
    zeros stays zero. Coefficients that let X, A or the polynomial grow beyond 10^9
    on the way overflow to NaN. Not differentiable."""
    native.refuse_tangents("newton_schulz", x)
    native.require_cuda(x)
    if x.dim() < 2:
        raise NativeError(f"newton_schulz: a matrix or a stack of matrices expected, got {tuple(x.shape)}")
    if torch.is_grad_enabled() and x.requires_grad:
        raise NativeError("newton_schulz: not differentiable (call it under torch.no_grad())")
    args = _ns_args("newton_schulz", x.dtype, steps, coefficients, eps)
    m, n = x.shape[-2:]
    stack = x.reshape(math.prod(x.shape[:-2]), m, n)
    if stack.numel() == 0:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    if (n > 1 and stack.stride(2) != 1) or (m > 1 and stack.stride(1) < n):
        stack = stack.contiguous()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    entry = native.NsEntry()
    entry.x, entry.ld_x, entry.stride_x = stack.data_ptr(), max(stack.stride(1), n), stack.stride(0)
    entry.out, entry.ld_out, entry.stride_out = out.data_ptr(), n, m * n
    entry.rows, entry.cols, entry.count = m, n, stack.shape[0]
    args.entries, args.n = ctypes.pointer(entry), 1
    with torch.cuda.device(x.device):
        workspace = _ns_workspace(args, x.device)
        native.invoke("cg_newton_schulz", ctypes.byref(args), native.stream_ptr(x.device))
    del workspace
    return out


class FusedMuon:
    """Muon over a flat buffer of matrices:

        m <- m + (1 - momentum) (g - m);  u = g + momentum (m - g)  (or m without nesterov)
        W <- (1 - lr weight_decay) W - lr sqrt(max(1, rows / cols)) newton_schulz(u)

    The momentum update, the norms and the split into half-precision planes are
    one pass each over the gradients, the Newton-Schulz products run batched
    over equal shapes, and the last product's epilogue applies the update to
    the weights. The products are those of newton_schulz on half-precision
    matrices: within 6e-6 of the update, 1e-5 on strongly decaying spectra (its
    fp32 form 1e-6 and 3e-6, torch's fp32 products 4e-6 and 5e-6). ``lr``, ``momentum`` and ``weight_decay`` may be changed
    between steps. Keeps a momentum buffer (4 bytes per parameter) and a
    workspace (about 8 bytes per parameter)."""

    def __init__(self, grads: FlatGradients, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.1, steps: int = 5,
                 coefficients: tuple[float, float, float] = NS_COEFFICIENTS, eps: float = 1e-7):
        if grads.flat.dtype != torch.float32:
            raise ValueError("FusedMuon: parameters must be float32")
        wrong = [tuple(p.shape) for p in grads.params if p.dim() != 2]
        if wrong:
            raise ValueError(f"FusedMuon: matrices expected, got parameters of shapes {wrong}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"FusedMuon: momentum {momentum} outside [0, 1)")
        self.grads = grads
        self._args = _ns_args("FusedMuon", torch.float32, steps, coefficients, eps)
        self.flat = _into_flat(grads)
        self.momentum_buffer = torch.zeros_like(self.flat)
        self.lr, self.momentum, self.nesterov, self.weight_decay = lr, momentum, nesterov, weight_decay
        self._entries = (native.NsEntry * len(grads.params))()
        for e, p, (offset, _) in zip(self._entries, grads.params, grads.offsets):
            e.rows, e.cols, e.count = p.shape[0], p.shape[1], 1
            e.ld_x = e.ld_out = e.ld_momentum = p.shape[1]
            e.x = grads.flat.data_ptr() + 4 * offset
            e.out = self.flat.data_ptr() + 4 * offset
            e.momentum = self.momentum_buffer.data_ptr() + 4 * offset
        self._args.entries = ctypes.cast(self._entries, ctypes.POINTER(native.NsEntry))
        self._args.n = len(grads.params)
        self._workspace: Tensor | None = None  # allocated by the first step

    @torch.no_grad()
    def step(self) -> None:
        args, device = self._args, self.flat.device
        native.require_cuda(self.flat)
        args.lr, args.momentum, args.weight_decay = self.lr, self.momentum, self.weight_decay
        args.nesterov = int(self.nesterov)
        with torch.cuda.device(device):
            if self._workspace is None:
                self._workspace = _ns_workspace(args, device)
            native.invoke("cg_muon_step", ctypes.byref(args), native.stream_ptr(device))
