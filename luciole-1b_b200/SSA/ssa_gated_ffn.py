"""Gated feed-forward over libssa_b200.so: both projections, the activation and the product in one
kernel, with the backward.

``ssa_gated_ffn(x, weight_gate_up)`` is ``silu(g) * u`` with ``g, u = (x @ weight_gate_up.T)
.chunk(2, -1)``. Only x and the weights are kept for the backward, which forms g and u again.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function

from . import _lib

__all__ = ["SSAGatedFFNFunc", "ssa_gated_ffn"]


def _problem(x, w):
    return _lib.SsaGatedFfn(_lib.DTYPE_CODES[x.dtype], _lib.int32(x.shape[0]),
                            _lib.int32(x.shape[1]), _lib.int32(w.shape[0] // 2), x.data_ptr(),
                            _lib.row_stride(x), w.data_ptr(), _lib.row_stride(w))


def _forward(inp, weight):
    """h and the matrices it was computed from."""
    dev = inp.device
    x = _lib.tma_matrix(inp if inp.dim() == 2 else inp.reshape(-1, inp.shape[-1]))
    w = _lib.tma_matrix(weight)
    f = w.shape[0] // 2
    h = torch.empty(*inp.shape[:-1], f, device=dev, dtype=inp.dtype)
    if x.shape[0]:
        prob = _problem(x, w)
        with _lib.device_guard(dev):
            rc = _lib.load().ssa_gated_ffn_fwd(ctypes.byref(prob), h.data_ptr(), f,
                                               _lib.stream_ptr(dev))
        _lib.check(rc)
    return h, x, w


class SSAGatedFFNFunc(Function):
    """h = silu(x Wg^T) * (x Wu^T); gradients of x and [Wg; Wu]."""

    @staticmethod
    def forward(ctx, inp, weight):
        h, x, w = _forward(inp, weight)
        ctx.save_for_backward(x, w)
        ctx.shape = inp.shape
        return h

    @staticmethod
    @_lib.first_order
    def backward(ctx, grad):
        x, w = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need_x else None
        dw = torch.empty(w.shape, device=w.device, dtype=w.dtype) if need_w else None
        if x.shape[0] == 0:
            if dw is not None:
                dw.zero_()
        elif need_x or need_w:
            lib = _lib.load()
            dh = grad.reshape(-1, w.shape[0] // 2)
            if dh.stride(1) != 1 or _lib.row_stride(dh) < dh.shape[1]:
                dh = dh.contiguous()
            prob = _problem(x, w)
            ws = _lib.workspace(lib.ssa_gated_ffn_bwd_workspace_size(ctypes.byref(prob)), x.device)
            with _lib.device_guard(x.device):
                rc = lib.ssa_gated_ffn_bwd(
                    ctypes.byref(prob), dh.data_ptr(), _lib.row_stride(dh),
                    dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None,
                    ws.data_ptr(), ws.numel(), _lib.stream_ptr(x.device))
            _lib.check(rc)
        return dx.view(ctx.shape) if need_x else None, dw


def ssa_gated_ffn(x, weight_gate_up):
    """``silu(x @ Wg.T) * (x @ Wu.T)`` for ``weight_gate_up = [Wg; Wu]`` of shape [2 F, H] (the
    weight of one linear layer whose output is chunked into gate and up).

    x [..., H]: fp16 or bf16 CUDA tensor, H a multiple of 8, F any size; the weight has x's dtype
    (layouts TMA cannot address are copied). Returns [..., F] in x's dtype. fp32 accumulation and
    activation, one rounding of h; in the backward one rounding of the pre-activations' gradients
    and one of the results, which are the same from run to run."""
    if not isinstance(x, torch.Tensor) or not isinstance(weight_gate_up, torch.Tensor):
        raise ValueError("x and weight_gate_up must be tensors")
    w = weight_gate_up
    if not (x.is_cuda and w.is_cuda):
        raise ValueError("x and weight_gate_up must be CUDA tensors (there is no CPU path)")
    if x.device != w.device:
        raise ValueError("x and weight_gate_up must be on one device")
    if x.dtype not in (torch.float16, torch.bfloat16) or w.dtype != x.dtype:
        raise ValueError(f"x and weight_gate_up must both be fp16 or both bf16, got {x.dtype} and "
                         f"{w.dtype}")
    if x.dim() < 1 or w.dim() != 2 or w.shape[1] != x.shape[-1] or w.shape[0] % 2 or not w.shape[0]:
        raise ValueError(f"weight_gate_up must be [2 F, H] for x [..., H], got {tuple(w.shape)} and "
                         f"{tuple(x.shape)}")
    if x.shape[-1] < 8 or x.shape[-1] % 8:
        raise ValueError(f"hidden size {x.shape[-1]} must be a positive multiple of 8")
    if _lib.differentiated(x, w):
        return SSAGatedFFNFunc.apply(x, w)
    return _forward(x, w)[0]
