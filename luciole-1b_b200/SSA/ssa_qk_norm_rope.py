"""Per-head norm and position rotation of queries and keys over libssa_b200.so, in one pass over the
packed qkv projection, with the backward.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function

from . import _lib

__all__ = ["SSAQKNormRopeFunc", "ssa_qk_norm_rope"]


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """`t` [.., D] if its last dimension is contiguous and its base and other strides are 16-byte aligned,
    else a copy in fresh storage."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t  # D is a multiple of 16
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
            s * t.element_size() % 16 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _tensor(t: torch.Tensor) -> _lib.SsaTensor:
    """[B, S, H, D] as the library's strided [B, H, S, D]; strides of extent 1 are never used."""
    (b, s, h, _), (sb, ss, sh, _) = t.shape, t.stride()
    return _lib.SsaTensor(t.data_ptr(), sb if b > 1 else 0, sh if h > 1 else 0, ss if s > 1 else 0)


def _problem(x, hq, hkv, cos, sin, pos, pos_stride, wq, wk, eps):
    """x [B, S, Hq + 2 Hkv, D]."""
    return _lib.SsaQkRope(
        _lib.DTYPE_CODES[x.dtype], _lib.int32(x.shape[0]), _lib.int32(x.shape[1]), _lib.int32(hq),
        _lib.int32(hkv), x.shape[3], _tensor(x), cos.data_ptr(), sin.data_ptr(),
        _lib.int32(cos.shape[0]), pos.data_ptr() if pos is not None else None,
        1 if pos is not None and pos.dtype == torch.int64 else 0, pos_stride,
        wq.data_ptr() if wq is not None else None, wk.data_ptr() if wk is not None else None,
        _lib.DTYPE_CODES[wq.dtype if wq is not None else x.dtype], eps)


def _forward(qkv, q_weight, k_weight, cos, sin, positions, hq, hkv, eps):
    """q, k, v, the tensors the backward needs, and the stride between sequences' positions."""
    d = cos.shape[1]
    lead = qkv.shape[:-1]
    heads = qkv.view(*lead, hq + 2 * hkv, d)
    x = _aligned(heads if len(lead) == 2 else heads.unsqueeze(0))
    cos, sin = _lib.table(cos), _lib.table(sin)
    pos, pos_stride = positions, 0
    if pos is not None:
        pos = pos.contiguous()
        pos_stride = lead[1] if pos.dim() == 2 else 0
    wq = q_weight.contiguous() if q_weight is not None else None
    wk = k_weight.contiguous() if k_weight is not None else None
    q = torch.empty(*lead, hq, d, device=qkv.device, dtype=qkv.dtype)
    k = torch.empty(*lead, hkv, d, device=qkv.device, dtype=qkv.dtype)
    if q.numel():
        prob = _problem(x, hq, hkv, cos, sin, pos, pos_stride, wq, wk, eps)
        with _lib.device_guard(qkv.device):
            rc = _lib.load().ssa_qk_rope_fwd(ctypes.byref(prob), q.data_ptr(), k.data_ptr(),
                                             _lib.stream_ptr(qkv.device))
        _lib.check(rc)
    return (q, k, heads.narrow(-2, hq + hkv, hkv)), (x, cos, sin, pos, wq, wk), pos_stride


class SSAQKNormRopeFunc(Function):
    """(q, k, v) of a packed qkv projection; gradients of qkv and the norm weights."""

    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, cos, sin, positions, hq, hkv, eps):
        out, saved, pos_stride = _forward(qkv, q_weight, k_weight, cos, sin, positions, hq, hkv, eps)
        # without the norm the rotation's gradient needs no x
        ctx.save_for_backward(saved[0] if q_weight is not None else None, *saved[1:])
        ctx.args = (hq, hkv, eps, pos_stride, qkv.shape)
        return out

    @staticmethod
    @_lib.first_order
    def backward(ctx, dq, dk, dv):
        x, cos, sin, pos, wq, wk = ctx.saved_tensors
        hq, hkv, eps, pos_stride, shape = ctx.args
        grads = [_aligned(g if len(shape) == 3 else g.unsqueeze(0)) for g in (dq, dk, dv)]
        dqkv = torch.empty(shape, device=dq.device, dtype=dq.dtype)
        dwq = torch.empty_like(wq) if wq is not None else None
        dwk = torch.empty_like(wk) if wk is not None else None
        if dqkv.numel():
            lib = _lib.load()
            # without the norm the projection is not read: dqkv stands in for its shape and address
            view = x if x is not None else dqkv.view(*grads[0].shape[:2], hq + 2 * hkv, cos.shape[1])
            prob = _problem(view, hq, hkv, cos, sin, pos, pos_stride, wq, wk, eps)
            ws = _lib.workspace(lib.ssa_qk_rope_bwd_workspace_size(ctypes.byref(prob)), dq.device)
            with _lib.device_guard(dq.device):
                rc = lib.ssa_qk_rope_bwd(
                    ctypes.byref(prob), *(_tensor(g) for g in grads), dqkv.data_ptr(),
                    dwq.data_ptr() if dwq is not None else None,
                    dwk.data_ptr() if dwk is not None else None, ws.data_ptr(), ws.numel(),
                    _lib.stream_ptr(dq.device))
            _lib.check(rc)
        elif dwq is not None:
            dwq.zero_()
            dwk.zero_()
        return dqkv, dwq, dwk, None, None, None, None, None, None


def ssa_qk_norm_rope(qkv, num_heads, num_kv_heads, cos, sin, q_weight=None, k_weight=None, eps=1e-5,
                     positions=None):
    """Queries, keys and values of a packed projection, with queries and keys normed per head and
    rotated: ``y = n * cos + rotate_half(n) * sin`` with ``n = x * rsqrt(mean(x^2) + eps) * weight``
    (or ``n = x`` without weights), in fp32 with one rounding.

    qkv: [B, S, (Hq + 2 Hkv) D] or packed [T, (Hq + 2 Hkv) D], fp32, fp16 or bf16 on CUDA, queries'
    heads first, then keys', then values'; D 16, 32, 64 or 128. cos, sin: fp32 [P, D] (``rope_tables``), which
    get no gradient.
    q_weight, k_weight: [D], both or neither, fp32 or of qkv's dtype. positions: None (row s of a
    sequence has position s), or int32 / int64 of shape [S], [B, S] or [T], an index into the tables;
    one outside them gives NaN (nothing is read out of range). Returns q [..., Hq, D], k [..., Hkv, D]
    and v [..., Hkv, D], the last a view of qkv. Layouts the kernels cannot address are copied."""
    if qkv is None or cos is None or sin is None:
        raise ValueError("qkv, cos and sin are required")
    for t in (qkv, cos, sin, q_weight, k_weight, positions):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError("qkv, cos, sin, the weights and positions must be tensors")
        if not t.is_cuda or t.get_device() != qkv.get_device():
            raise ValueError("all tensors must be CUDA tensors (there is no CPU path) on one device")
    if qkv.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"unsupported dtype {qkv.dtype}")
    hq, hkv = int(num_heads), int(num_kv_heads)
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 \
            or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be fp32 [P, D] tables of one shape")
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise ValueError("cos and sin are tables without a gradient: detach them")
    d = cos.shape[1]
    if d not in (16, 32, 64, 128):
        raise ValueError(f"head dim D={d} not supported (16, 32, 64, 128)")
    if hq < 1 or hkv < 1 or qkv.dim() not in (2, 3) or qkv.shape[-1] != (hq + 2 * hkv) * d:
        raise ValueError(f"qkv {tuple(qkv.shape)} must be [B, S, C] or [T, C] with C = "
                         f"(Hq + 2 Hkv) D = {(hq + 2 * hkv) * d}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight come together or not at all")
    if q_weight is not None and (
            q_weight.shape != (d,) or k_weight.shape != (d,) or q_weight.dtype != k_weight.dtype
            or q_weight.dtype not in (torch.float32, qkv.dtype)):
        raise ValueError(f"q_weight and k_weight must be [{d}], fp32 or {qkv.dtype}")
    lead = qkv.shape[:-1]
    if positions is None:
        if lead[-1] > cos.shape[0]:
            raise ValueError(f"{lead[-1]} rows, but tables of {cos.shape[0]} positions")
    else:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if tuple(positions.shape) not in ((lead[-1],), tuple(lead)):
            raise ValueError(f"positions {tuple(positions.shape)} do not fit rows {tuple(lead)}")
        if cos.shape[0] < 1:
            raise ValueError("empty cos / sin tables")
    if _lib.differentiated(qkv, q_weight, k_weight) or _lib.has_tangent((cos, sin)):
        return SSAQKNormRopeFunc.apply(qkv, q_weight, k_weight, cos, sin, positions, hq, hkv,
                                       float(eps))
    return _forward(qkv, q_weight, k_weight, cos, sin, positions, hq, hkv, float(eps))[0]
