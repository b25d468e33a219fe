"""Order on a stream between the kernels that start programmatically.

A kernel that lets its dependents start before it has itself waited for the kernel ahead hands on a
start that waits for nothing: a dependent that touches memory ahead of its own wait (the attention
backward reads K and V and writes partial sums there) can then run beside the kernel before the last.
On the CPU the sources are read for that order; on the GPU each pair of kernels that it concerns runs
back to back and must give what it gives with a synchronisation between."""

import re
from pathlib import Path

import pytest
import torch

CSRC = Path(__file__).resolve().parent.parent / "luciole-1b_b200" / "csrc"


def _kernels(text):
    """(name, body) of every __global__ function."""
    text = re.sub(r"//[^\n]*", "", text)
    for part in re.split(r"__global__", text)[1:]:
        name = re.search(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\s*\([^)]*\)", "", part)).group(1)
        depth, start = 0, part.index("{")
        for i in range(start, len(part)):
            depth += (part[i] == "{") - (part[i] == "}")
            if depth == 0:
                break
        yield name, part[start:i]


def test_dependents_start_after_the_kernel_has_waited():
    seen = 0
    for f in sorted(CSRC.glob("*.cu*")):
        for name, body in _kernels(f.read_text()):
            go = body.find("griddep_launch_dependents(")
            if go >= 0:
                seen += 1
                assert 0 <= body.find("griddep_wait(") < go, (f.name, name)
    assert seen >= 10


def _attention(dev, dtype=torch.bfloat16, b=2, s=2048, hq=16, hkv=4, d=64):
    """A packed projection with its rotation tables, the attention's forward on it, and a gradient."""
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    from SSA.ssa_triton_kernel import ssa_flash_attn_forward
    from luciole_train import rope_tables
    g = torch.Generator(device=dev).manual_seed(3)
    qkv = torch.randn(b, s, (hq + 2 * hkv) * d, generator=g, device=dev).to(dtype)
    cos, sin = rope_tables(s, d, 1e4, dev)
    n, bb = torch.full((hq,), 0.43, device=dev), torch.tensor(0.8, device=dev)

    def rotate():
        return [t.transpose(1, 2) for t in ssa_qk_norm_rope(qkv, hq, hkv, cos, sin)]

    q, k, v = rotate()
    out, lse = ssa_flash_attn_forward(q, k, v, d ** -0.5, n, bb, True)
    dout = torch.randn(out.shape, generator=g, device=dev).to(dtype)
    return rotate, (out, dout, lse), (d ** -0.5, n, bb)


def _backward(q, k, v, rest, par, deterministic):
    from SSA.ssa_triton_kernel import ssa_flash_attn_backward
    out, dout, lse = rest
    return ssa_flash_attn_backward(q, k, v, out, dout, lse, *par, True, deterministic=deterministic)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_rotation_directly_before_the_attention_backward(cuda_device, d):
    """Queries and keys formed again (as under recomputation) right before the backward that reads
    them; the blocks they land in held NaN before."""
    rotate, rest, par = _attention(cuda_device, d=d)
    want = _backward(*rotate(), rest, par, True)
    torch.cuda.synchronize()
    for _ in range(10):
        q, k, _ = rotate()
        nan = [torch.full_like(t, float("nan")) for t in (q, k)]
        del q, k, nan
        torch.cuda.synchronize()
        got = _backward(*rotate(), rest, par, True)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_gradient_products_directly_before_a_deterministic_attention_backward(cuda_device):
    """The feed-forward's backward frees its workspace, from which the attention's backward takes its
    own: neither's results may change by following the other at once."""
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    rotate, rest, par = _attention(cuda_device)
    qkv = rotate()
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = torch.randn(2048, 1024, generator=g, device=cuda_device).bfloat16().requires_grad_(True)
    w = (torch.randn(5632, 1024, generator=g, device=cuda_device) / 32).bfloat16().requires_grad_(True)
    dh = torch.randn(2048, 2816, generator=g, device=cuda_device).bfloat16()

    def ffn():
        return torch.autograd.grad(ssa_gated_ffn(x, w), (x, w), dh)

    want = [*ffn()]
    torch.cuda.synchronize()
    want += _backward(*qkv, rest, par, True)
    torch.cuda.synchronize()
    for _ in range(10):
        got = [*ffn(), *_backward(*qkv, rest, par, True)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        del got
