"""
Refusals of the half-precision layer's C entry points, without a GPU: an
activation code that is none of theirs is an error, not an identity. The calls
run on a thread of their own: the text of the last error is kept per thread.
"""

from __future__ import annotations

import ctypes
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from create_graph_b200 import native

X = torch.zeros(8, 8, dtype=torch.bfloat16)


def act_grad(act):
    args = native.ActGradArgs()
    args.rows = args.cols = args.ld_gy = args.ld_z = args.ld_gz = 8
    args.gy = args.z = args.gz = X.data_ptr()
    args.act, args.dtype = act, native.BF16
    return native.load_library().cg_act_grad_half(ctypes.byref(args), None)


def act_grad2(act):
    p = X.data_ptr()
    return native.load_library().cg_act_grad2_half(p, None, p, p, p, p, 8, 8, act, native.BF16, None)


def backward(act):
    args = native.LinearBackwardArgs()
    args.m = args.n = args.k = args.ld_gy = args.ld_z = args.ld_gz = args.ld_x = args.ld_w = 8
    args.gy = args.z = args.gz = args.x = args.w = X.data_ptr()
    args.act, args.dtype = act, native.BF16
    return native.load_library().cg_linear_half_backward(ctypes.byref(args), None)


@pytest.mark.parametrize("entry", [act_grad, act_grad2, backward])
@pytest.mark.parametrize("act", [native.ACT_SILU_GRAD, native.ACT_ADD, 6, -1])
def test_unknown_activations_are_refused(entry, act):
    with ThreadPoolExecutor(1) as thread:
        assert thread.submit(entry, act).result() != 0
        assert f"bad act {act}" in thread.submit(native.load_library().cg_last_error).result().decode()
