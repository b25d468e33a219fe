"""Global gradient norm and clipping over libssa_b200.so.

``ssa_grad_norm(grads)`` is the 2-norm over a list of tensors; ``ssa_clip_grad_norm(grads,
max_norm)`` scales them by ``min(1, max_norm / (norm + 1e-6))`` in place, or into the tensors of
``out`` (fp32 for an optimizer's master gradients: the conversion and the clipping are one pass).
Neither synchronises with the host.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib

__all__ = ["ssa_grad_norm", "ssa_clip_grad_norm"]


def _check_list(ts, what, device=None, dtype=None):
    """A list of CUDA tensors of one device and one floating dtype."""
    ts = list(ts)
    for t in ts:
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise ValueError(f"{what} must be dense tensors")
        device = t.device if device is None else device
        dtype = t.dtype if dtype is None else dtype
        if t.device != device or t.dtype != dtype:
            raise ValueError(f"{what} must be on one device and of one dtype, got {t.dtype} on "
                             f"{t.device} beside {dtype} on {device}")
    if ts and device.type != "cuda":
        raise ValueError(f"{what} must be CUDA tensors (there is no CPU path)")
    if ts and dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"{what} must be fp32, fp16 or bf16, got {dtype}")
    return ts


def _overlap(ptrs, sizes, item):
    """Whether two of the (contiguous) tensors share memory."""
    used = sizes > 0
    order = np.argsort(ptrs[used], kind="stable")
    start, nbytes = ptrs[used][order], sizes[used][order] * item
    return bool((start[1:] < start[:-1] + nbytes[:-1]).any())


def _arrays(ts):
    n = len(ts)
    return (np.fromiter((t.data_ptr() for t in ts), np.int64, n),
            np.fromiter((t.numel() for t in ts), np.int64, n))


def _list(ptrs, sizes, dtype, outs=None, out_dtype=None):
    return _lib.SsaGradList(
        _lib.DTYPE_CODES[dtype], len(sizes), ptrs.ctypes.data, sizes.ctypes.data,
        outs.ctypes.data if outs is not None else None,
        _lib.DTYPE_CODES[out_dtype if out_dtype is not None else dtype])


def ssa_grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """The 2-norm over all elements of a list of tensors (fp32, fp16 or bf16, one dtype, one CUDA
    device), as an fp32 scalar on their device. Squares are summed in 64 bits in a fixed order;
    infinities and NaN in a gradient come through. An empty list gives 0 on the current device."""
    grads = _check_list(grads, "grads")
    if not grads:
        return torch.zeros((), device="cuda")
    dev = grads[0].device
    held = [t if t.is_contiguous() else t.contiguous() for t in grads]
    ptrs, sizes = _arrays(held)
    lib = _lib.load()
    lst = _list(ptrs, sizes, grads[0].dtype)
    norm = torch.empty((), device=dev, dtype=torch.float32)
    ws = _lib.workspace(lib.ssa_grad_clip_workspace_size(ctypes.byref(lst)), dev)
    with _lib.device_guard(dev):
        rc = lib.ssa_grad_norm(ctypes.byref(lst), norm.data_ptr(), ws.data_ptr(), ws.numel(),
                               _lib.stream_ptr(dev))
    _lib.check(rc)
    return norm


@torch.no_grad()
def ssa_clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float,
                       out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scale ``grads`` so that their 2-norm is at most ``max_norm``; returns the norm before that
    (fp32 scalar on their device).

    Every element is multiplied by ``min(1, max_norm / (norm + 1e-6))`` in fp32 and rounded once: in
    place, or, with ``out``, into contiguous tensors of the same sizes that are fp32 or of the
    gradients' dtype (``grads`` then stay as they are). As with torch's clipping, a NaN norm makes
    every gradient NaN and an infinite one makes the finite ones 0. grads: one dtype (fp32, fp16,
    bf16), one CUDA device; tensors that are written must not share memory."""
    grads = _check_list(grads, "grads")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be at least 0, got {max_norm}")
    if out is not None:
        out = _check_list(out, "out", grads[0].device if grads else None)
        if len(out) != len(grads):
            raise ValueError(f"out has {len(out)} tensors for {len(grads)} gradients")
        for g, o in zip(grads, out):
            if g.shape != o.shape:
                raise ValueError(f"out {tuple(o.shape)} does not have its gradient's shape "
                                 f"{tuple(g.shape)}")
            if not o.is_contiguous():
                raise ValueError("out must be contiguous")
        if out and out[0].dtype not in (torch.float32, grads[0].dtype):
            raise ValueError(f"out must be fp32 or of the gradients' dtype, got {out[0].dtype}")
    if not grads:
        return torch.zeros((), device="cuda")
    dev, dtype = grads[0].device, grads[0].dtype
    held = [t if t.is_contiguous() else t.contiguous() for t in grads]
    ptrs, sizes = _arrays(held)
    optrs, out_dtype = None, dtype
    if out is None:
        strided = [(g, h) for g, h in zip(grads, held) if g is not h]
        item = held[0].element_size()
        if _overlap(ptrs, sizes, item) or any(n > 1 and s == 0 for g, _ in strided
                                              for n, s in zip(g.shape, g.stride())):
            raise ValueError("gradients that are scaled in place must not share memory")
    else:
        strided = []
        optrs, _ = _arrays(out)
        out_dtype = out[0].dtype
        item = out[0].element_size()
        both = np.concatenate([ptrs, optrs])
        nbytes = np.concatenate([sizes * held[0].element_size(), sizes * item])
        same = item == held[0].element_size() and bool((ptrs == optrs).all())
        if _overlap(optrs, sizes, item) or (not same and _overlap_between(both, nbytes, len(out))):
            raise ValueError("out must not share memory, neither within itself nor with grads")
    lib = _lib.load()
    lst = _list(ptrs, sizes, dtype, optrs, out_dtype)
    norm = torch.empty((), device=dev, dtype=torch.float32)
    ws = _lib.workspace(lib.ssa_grad_clip_workspace_size(ctypes.byref(lst)), dev)
    with _lib.device_guard(dev):
        rc = lib.ssa_grad_clip(ctypes.byref(lst), max_norm, norm.data_ptr(), ws.data_ptr(),
                               ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc)
    torch.autograd.graph.increment_version(
        [t for t in (held if out is None else out) if not t.is_inference()])
    for g, h in strided:
        g.copy_(h)
    return norm


def _overlap_between(ptrs, nbytes, n):
    """Whether one of the last n ranges meets one of the others (which may share among themselves)."""
    start, end = ptrs[:-n], ptrs[:-n] + nbytes[:-n]
    used = nbytes[-n:] > 0
    order = np.argsort(ptrs[-n:][used], kind="stable")
    os_, oe = ptrs[-n:][used][order], (ptrs[-n:] + nbytes[-n:])[used][order]
    at = np.searchsorted(os_, end, side="left")  # outputs that begin before a gradient ends
    top = np.concatenate([[0], np.maximum.accumulate(oe)])
    return bool(((top[at] > start) & (nbytes[:-n] > 0)).any())
