"""Cross entropy of a linear head over libssa_b200.so, without the logits.

``ssa_linear_cross_entropy(hidden, weight, targets)`` is
``cross_entropy(hidden @ weight.T, targets)``: the logits stay on the chip in fp32, the backward
forms them again per piece of the vocabulary, and neither pass holds a [tokens, vocab] matrix.

The backward's workspace: one 16-bit piece of the logits' gradient (with reduction "none" two), up to
256 MiB or 1024 columns, whichever is more; a 16-bit copy of the hidden states; and where there are
several pieces, or dx's contraction is split, their fp32 gradient once per split.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function

from . import _lib

__all__ = ["SSALinearCrossEntropyFunc", "ssa_linear_cross_entropy"]

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _problem(x, w, t, ignore_index, reduction):
    return _lib.SsaLinearCe(_lib.DTYPE_CODES[x.dtype], _lib.int32(x.shape[0]),
                            _lib.int32(x.shape[1]), _lib.int32(w.shape[0]), x.data_ptr(),
                            _lib.row_stride(x), w.data_ptr(), _lib.row_stride(w), t.data_ptr(),
                            ignore_index, reduction)


def _forward(hidden, weight, targets, ignore_index, code):
    """The loss, and what the backward needs: x, w, targets, the rows' lse, the rows counted."""
    dev = hidden.device
    x = _lib.tma_matrix(hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1]))
    w = _lib.tma_matrix(weight)
    t = targets.reshape(-1).to(torch.int64).contiguous()
    n = x.shape[0]
    stats = torch.empty(n + 1, device=dev, dtype=torch.float32)  # lse of the rows, their count
    if n == 0:
        loss = stats.new_empty(targets.shape) if code == 0 else \
            stats.new_full((), float("nan") if code == 1 else 0.0)
    else:
        loss = torch.empty(targets.shape if code == 0 else (), device=dev, dtype=torch.float32)
        lib = _lib.load()
        prob = _problem(x, w, t, ignore_index, code)
        ws = _lib.workspace(lib.ssa_linear_ce_fwd_workspace_size(ctypes.byref(prob)), dev)
        lse = stats.data_ptr()
        with _lib.device_guard(dev):
            rc = lib.ssa_linear_ce_fwd(ctypes.byref(prob), loss.data_ptr(), lse, lse + 4 * n,
                                       ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
        _lib.check(rc)
    return loss, x, w, t, stats


class SSALinearCrossEntropyFunc(Function):
    """loss = reduce(logsumexp(x W^T) - (x W^T)[target]); gradients of x and W."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        code = _REDUCTIONS[reduction]
        loss, *saved = _forward(hidden, weight, targets, ignore_index, code)
        ctx.save_for_backward(*saved)
        ctx.args = (ignore_index, code, hidden.shape)
        return loss

    @staticmethod
    @_lib.first_order
    def backward(ctx, grad_loss):
        x, w, t, stats = ctx.saved_tensors
        ignore_index, code, shape = ctx.args
        need_x, need_w = ctx.needs_input_grad[:2]
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need_x else None
        dw = torch.empty(w.shape, device=w.device, dtype=w.dtype) if need_w else None
        if x.shape[0] == 0:
            if dw is not None:
                dw.zero_()
        elif need_x or need_w:
            lib = _lib.load()
            g = grad_loss.reshape(-1).to(torch.float32).contiguous()
            prob = _problem(x, w, t, ignore_index, code)
            ws = _lib.workspace(lib.ssa_linear_ce_bwd_workspace_size(ctypes.byref(prob)), x.device)
            lse = stats.data_ptr()
            with _lib.device_guard(x.device):
                rc = lib.ssa_linear_ce_bwd(
                    ctypes.byref(prob), lse, lse + 4 * x.shape[0], g.data_ptr(),
                    dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None,
                    ws.data_ptr(), ws.numel(), _lib.stream_ptr(x.device))
            _lib.check(rc)
        return dx.view(shape) if need_x else None, dw, None, None, None


def ssa_linear_cross_entropy(hidden, weight, targets, ignore_index=-100, reduction="mean"):
    """Cross entropy of the logits ``hidden @ weight.T`` against ``targets``.

    hidden [..., H] and weight [V, H]: fp16 or bf16 CUDA tensors of one dtype, H a multiple of 8
    (layouts TMA cannot address are copied). targets [...]: int64 or int32; a row whose target is
    ``ignore_index`` has loss 0 and no gradient, and a target outside [0, V) makes that row's loss
    and the gradients NaN (nothing is read out of range). reduction: "mean" (over the rows that are
    not ignored; NaN if there are none), "sum" or "none". Returns fp32; gradients come in the
    inputs' dtype and are the same from run to run."""
    if not isinstance(hidden, torch.Tensor) or not isinstance(weight, torch.Tensor) \
            or not isinstance(targets, torch.Tensor):
        raise ValueError("hidden, weight and targets must be tensors")
    if not (hidden.is_cuda and weight.is_cuda and targets.is_cuda):
        raise ValueError("hidden, weight and targets must be CUDA tensors (there is no CPU path)")
    if hidden.device != weight.device or hidden.device != targets.device:
        raise ValueError("hidden, weight and targets must be on one device")
    if hidden.dtype not in (torch.float16, torch.bfloat16) or weight.dtype != hidden.dtype:
        raise ValueError(f"hidden and weight must both be fp16 or both bf16, got {hidden.dtype} and "
                         f"{weight.dtype}")
    if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1]:
        raise ValueError(f"shape mismatch hidden={tuple(hidden.shape)} weight={tuple(weight.shape)}")
    if weight.shape[0] < 1 or weight.shape[1] < 8 or weight.shape[1] % 8:
        raise ValueError(f"hidden size {weight.shape[1]} must be a positive multiple of 8, and the "
                         "vocabulary not empty")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} must have hidden's leading shape "
                         f"{tuple(hidden.shape[:-1])}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets must be int64 or int32, got {targets.dtype}")
    if not -(1 << 63) <= int(ignore_index) < 1 << 63:
        raise ValueError(f"ignore_index {ignore_index} does not fit 64 bits")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if _lib.differentiated(hidden, weight):
        return SSALinearCrossEntropyFunc.apply(hidden, weight, targets, int(ignore_index), reduction)
    return _forward(hidden, weight, targets, int(ignore_index), _REDUCTIONS[reduction])[0]
