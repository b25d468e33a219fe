"""Global gradient norm and clipping over libssa_b200.so.

``ssa_grad_norm(grads)`` is the 2-norm over a list of tensors; ``ssa_clip_grad_norm(grads,
max_norm)`` scales them by ``min(1, max_norm / (norm + 1e-6))`` in place, or into the tensors of
``out`` (fp32 for an optimizer's master gradients: the conversion and the clipping are one pass).
Neither synchronises with the host.
"""

from __future__ import annotations

import ctypes
from array import array
from typing import Optional, Sequence

import torch

from . import _lib

__all__ = ["ssa_grad_norm", "ssa_clip_grad_norm"]


def _check_list(ts, what, device=None):
    """A list of dense CUDA tensors of one device and one floating dtype."""
    ts = list(ts)
    if not all([isinstance(t, torch.Tensor) and t.layout is torch.strided for t in ts]):
        raise ValueError(f"{what} must be dense tensors")
    dtypes = {t.dtype for t in ts}
    devices = {t.get_device() for t in ts}  # -1: the CPU
    if device is not None and ts:
        devices.add(device)
    if len(dtypes) > 1 or len(devices) > 1:
        raise ValueError(f"{what} must be on one device and of one dtype, got {dtypes} on {devices}")
    if ts and not ts[0].is_cuda:
        raise ValueError(f"{what} must be CUDA tensors (there is no CPU path)")
    if ts and ts[0].dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"{what} must be fp32, fp16 or bf16, got {ts[0].dtype}")
    if _lib.has_tangent(ts):
        raise NotImplementedError(f"{what} carry forward-mode tangents, which are not followed")
    return ts


def _pointers(ts):
    return array("q", [t.data_ptr() for t in ts])


def _run(grads, held, max_norm=None, out=None):
    """The norm (max_norm None) or the clipping of the contiguous tensors `held`."""
    dev = grads[0].device
    ptrs, sizes = _pointers(held), array("q", [t.numel() for t in held])
    optrs = _pointers(out) if out is not None else None
    lst = _lib.SsaGradList(
        _lib.DTYPE_CODES[grads[0].dtype], len(sizes), ptrs.buffer_info()[0], sizes.buffer_info()[0],
        optrs.buffer_info()[0] if out is not None else None,
        _lib.DTYPE_CODES[(out or grads)[0].dtype])
    lib = _lib.load()
    norm = torch.empty((), device=dev, dtype=torch.float32)
    ws = _lib.workspace(lib.ssa_grad_clip_workspace_size(ctypes.byref(lst)), dev)
    with _lib.device_guard(dev):
        st = _lib.stream_ptr(dev)
        if max_norm is None:
            rc = lib.ssa_grad_norm(ctypes.byref(lst), norm.data_ptr(), ws.data_ptr(), ws.numel(), st)
        else:
            rc = lib.ssa_grad_clip(ctypes.byref(lst), max_norm, norm.data_ptr(), ws.data_ptr(),
                                   ws.numel(), st)
    _lib.check(rc)
    return norm


def _contiguous(grads):
    if all([t.is_contiguous() for t in grads]):
        return grads
    return [t if t.is_contiguous() else t.detach().contiguous() for t in grads]


def ssa_grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """The 2-norm over all elements of a list of tensors (fp32, fp16 or bf16, one dtype, one CUDA
    device), as an fp32 scalar on their device. Squares are summed in 64 bits in a fixed order;
    infinities and NaN in a gradient come through. An empty list gives 0 on the current device.

    The norm takes no part in autograd: gradients that have a graph of their own (create_graph=True) are
    refused unless detached or under torch.no_grad()."""
    grads = _check_list(grads, "grads")
    if torch.is_grad_enabled() and any([t.grad_fn is not None for t in grads]):
        raise ValueError("the norm is not differentiable: detach gradients made with create_graph, or "
                         "call it under torch.no_grad()")
    return _run(grads, _contiguous(grads)) if grads else torch.zeros((), device="cuda")


def ssa_clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float,
                       out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scale ``grads`` so that their 2-norm is at most ``max_norm``; returns the norm before that
    (fp32 scalar on their device).

    Every element is multiplied by ``min(1, max_norm / (norm + 1e-6))`` in fp32 and rounded once: in
    place, or, with ``out``, into contiguous tensors of the same sizes that are fp32 or of the
    gradients' dtype (``grads`` then stay as they are). As with torch's clipping, a NaN norm makes
    every gradient NaN and an infinite one makes the finite ones 0, and autograd does not record the
    scaling: the norm and ``out`` are without a graph. grads: one dtype (fp32, fp16,
    bf16), one CUDA device; tensors that are written must not share memory, with one another or
    with gradients that are read."""
    grads = _check_list(grads, "grads")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be at least 0, got {max_norm}")
    if out is not None:
        out = _check_list(out, "out", grads[0].get_device() if grads else None)
        if len(out) != len(grads):
            raise ValueError(f"out has {len(out)} tensors for {len(grads)} gradients")
        if [o.shape for o in out] != [g.shape for g in grads]:
            raise ValueError("out must have the gradients' shapes")
        if not all([o.is_contiguous() for o in out]):
            raise ValueError("out must be contiguous")
        if out and out[0].dtype not in (torch.float32, grads[0].dtype):
            raise ValueError(f"out must be fp32 or of the gradients' dtype, got {out[0].dtype}")
    if not grads:
        return torch.zeros((), device="cuda")
    held = _contiguous(grads)
    back = [] if out is not None or held is grads else \
        [(g, h) for g, h in zip(grads, held) if g is not h]
    if any(n > 1 and s == 0 for g, _ in back for n, s in zip(g.shape, g.stride())):
        raise ValueError("gradients that are scaled in place must not share memory")
    norm = _run(grads, held, max_norm, out)
    torch.autograd.graph.increment_version(
        [t for t in (held if out is None else out) if not t.is_inference()])
    if back:
        with torch.no_grad():
            for g, h in back:
                g.copy_(h)
    return norm
