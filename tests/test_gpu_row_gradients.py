"""Linear cross entropy with one gradient per row (reduction "none"): a row's gradient depends on its own
factor alone, and every term of both gradients is rounded once before the sums.

Bounds, as in the tests of the operator, with u = eps / 2 and DL the error of a logit: an entry of
d = p - [v = t] is off by (u + 2 DL + 2^-16) |d|, in fp16 by at least half a subnormal step of its scale
2^14 (2^-25 2^-14 = 2^-39); the target's carries p's error, 2 DL, as well. dx multiplies the sum of d W
by the row's gradient in fp32 and rounds once. dW's terms are d times grad_r / max |grad|, rounded once
for the product, the same subnormal step then being one of max |grad|; x enters as it is."""

import math

import pytest
import torch

from test_gpu_linear_ce import _data

pytestmark = pytest.mark.gpu


def _check(x, w, t, grad):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = ssa_linear_cross_entropy(xl, wl, t, reduction="none")
    gx, gw = torch.autograd.grad(loss, (xl, wl), grad)
    X, W, G = x.double(), w.double(), torch.where(t == -100, 0.0, grad.double())
    at = t.clamp(min=0)
    rows = torch.arange(len(t), device=t.device)
    d = torch.softmax(X @ W.t(), 1)
    d[rows, at] -= 1.0
    d[t == -100] = 0.0
    u = torch.finfo(x.dtype).eps / 2
    dl = (x.shape[1] / 8 + 8) * 2.0 ** -23 * float((X.abs() @ W.abs().t()).max())
    e = u + 2 * dl + 2.0 ** -16
    sub = 2.0 ** -39 if x.dtype == torch.float16 else 0.0
    D = e * d.abs() + sub
    D[rows, at] += 2 * dl
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    dx, dw = G[:, None] * (d @ W), (G[:, None] * d).t() @ X
    bx = G.abs()[:, None] * (D @ W.abs()) + u * dx.abs() + tiny
    bw = (G.abs()[:, None] * (D - sub) + G.abs().max() * sub).t() @ X.abs() + u * dw.abs() + tiny
    for name, got, want, b in (("dx", gx, dx, bx), ("dw", gw, dw, bw)):
        # a result of at least the type's largest number and half a step rounds to infinity: 65,520 in
        # fp16 (a gradient of 4e4 times hidden states of 2 and more)
        over = want.abs() + b >= torch.finfo(x.dtype).max * (1 + u / 2)
        inf = over & got.isinf() & (got.sign() == want.sign())
        off = torch.where(inf, 0.0, (got.double() - want).abs())
        assert (off <= b).all(), (name, int((off > b).sum()), float((off / b).max()))
    return gx, gw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [999, 50257])
def test_gradients_of_very_different_size(cuda_device, dtype, v):
    """Ratios of up to 4 million between rows, in a vocabulary whose probabilities are then small."""
    x, w, t = _data(48, 128, v, dtype, 71, 0.1, cuda_device)
    grad = torch.logspace(-10, 12, 48, base=2.0, device=cuda_device)
    _check(x, w, t, grad)
    _check(x, w, t, grad * torch.tensor([1.0, -1.0], device=cuda_device).repeat(24))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 3, 130])
def test_terms_are_rounded_once(cuda_device, dtype, n):
    """Few terms a sum: a second rounding of a term shows."""
    x, w, t = _data(n, 256, 4001, dtype, 73, 0.0, cuda_device)
    for seed in range(3):
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        _check(x, w, t, torch.rand(n, generator=g, device=cuda_device) + 0.5)


def test_a_row_does_not_see_the_others_gradients(cuda_device):
    x, w, t = _data(64, 128, 20011, torch.float16, 79, 0.1, cuda_device)
    grad = torch.rand(64, device=cuda_device) + 0.5
    gx, _ = _check(x, w, t, grad)
    other = grad.clone()
    other[1::2] *= 3.0e4
    assert torch.equal(_check(x, w, t, other)[0][::2], gx[::2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_equal_gradients_are_as_a_sum(cuda_device, dtype):
    """Whatever the common factor is: no rounding of its own on every row."""
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(300, 128, 5003, dtype, 83, 0.1, cuda_device)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    c = torch.full((), 0.3, device=cuda_device)
    a = torch.autograd.grad(ssa_linear_cross_entropy(xl, wl, t, reduction="sum"), (xl, wl), c)
    b = torch.autograd.grad(ssa_linear_cross_entropy(xl, wl, t, reduction="none"), (xl, wl),
                            c.expand(300))
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_gradients_that_are_zero_infinite_or_nan(cuda_device):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(40, 64, 700, torch.bfloat16, 89, 0.0, cuda_device)
    grad = torch.ones(40, device=cuda_device)
    grad[3] = 0.0
    gx, gw = _check(x, w, t, grad)
    assert not gx[3].any()
    for bad in (float("inf"), float("nan")):
        grad[5] = bad
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = ssa_linear_cross_entropy(xl, wl, t, reduction="none")
        hx, hw = torch.autograd.grad(loss, (xl, wl), grad)
        keep = torch.arange(40, device=cuda_device) != 5
        assert torch.equal(hx[keep], gx[keep])
        assert not hx[5].isfinite().any() and not hw.isfinite().any()
    skip = t.clone()
    skip[5] = -100  # an ignored row's gradient reaches nothing
    loss = ssa_linear_cross_entropy(xl, wl, skip, reduction="none")
    hx, hw = torch.autograd.grad(loss, (xl, wl), grad)
    assert torch.equal(hx[keep], gx[keep]) and not hx[5].any() and hw.isfinite().all()
    out = t.clone()
    out[3] = 700  # no such id: NaN, also under a gradient of 0
    loss = ssa_linear_cross_entropy(xl, wl, out, reduction="none")
    hx, hw = torch.autograd.grad(loss, (xl, wl), torch.where(keep, grad, 1.0))
    assert hx[3].isnan().all() and hw.isnan().all()


@pytest.mark.parametrize("which", ["x", "w"])
def test_only_one_gradient(cuda_device, which):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(300, 128, 9001, torch.bfloat16, 97, 0.1, cuda_device)
    grad = torch.rand(300, device=cuda_device) + 0.5
    gx, gw = _check(x, w, t, grad)
    xl, wl = x.clone(), w.clone()
    (xl if which == "x" else wl).requires_grad_(True)
    loss = ssa_linear_cross_entropy(xl, wl, t, reduction="none")
    got, = torch.autograd.grad(loss, xl if which == "x" else wl, grad)
    assert torch.equal(got, gx if which == "x" else gw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_several_pieces(cuda_device, dtype):
    """20,000 rows: the vocabulary in several pieces, both gradients summed or stored by piece."""
    x, w, t = _data(20000, 64, 9007, dtype, 101, 0.1, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(7)
    _check(x, w, t, torch.rand(20000, generator=g, device=cuda_device) + 0.5)
