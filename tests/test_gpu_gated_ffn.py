"""Gated feed-forward (SSA.ssa_gated_ffn) against the same formulas in 64 bits.

Bounds. The pre-activations are fp32 sums of exact products, off by at most
DL = (H / 8 + 8) 2^-23 sum |x||w| (H / 16 matrix instructions of a few fp32 steps each); silu' is at
most 1.1 and silu'' at most 0.5 in magnitude. h is then off by DL (1.1 |u| + |silu(g)|) and one
rounding u = eps / 2. The gradient d = [dg | du] is off by DL |dh| (0.5 |u| + 2.2) and one rounding,
the sums over it run in fp32, and the results are rounded once. 2^-18 relative covers the
exponential's and reciprocal's approximations and the fp32 sums."""

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _data(n, h, f, dtype, seed, dev, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, h, generator=g).to(dtype).to(dev)
    w = (torch.randn(2 * f, h, generator=g) * (scale / math.sqrt(h))).to(dtype).to(dev)
    dh = torch.randn(n, f, generator=g).to(dtype).to(dev)
    return x, w, dh


def _reference(x, w, dh):
    X, W, H = x.double(), w.double(), dh.double()
    f = W.shape[0] // 2
    g, u = X @ W[:f].t(), X @ W[f:].t()
    s = torch.sigmoid(g)
    silu = g * s
    h = silu * u
    r = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    dl = (x.shape[1] / 8 + 8) * 2.0 ** -23 * float((X.abs() @ W.abs().t()).max())
    e = 2.0 ** -18
    bh = dl * (1.1 * u.abs() + silu.abs()) + (r + e) * h.abs() + dl * dl + tiny
    d = torch.cat([H * u * s * (1 + g * (1 - s)), H * silu], 1)
    bd = dl * torch.cat([H.abs() * (0.5 * u.abs() + 2.2)] * 2, 1) + (r + e) * d.abs() + tiny
    dx, dw = d @ W, d.t() @ X
    bdx = bd @ W.abs() + r * dx.abs() + e * (d.abs() @ W.abs()) + tiny
    bdw = bd.t() @ X.abs() + r * dw.abs() + e * (d.t().abs() @ X.abs()) + tiny
    return (h, dx, dw), (bh, bdx, bdw)


def _check(x, w, dh):
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    h = ssa_gated_ffn(xl, wl)
    gx, gw = torch.autograd.grad(h, (xl, wl), dh)
    want, bounds = _reference(x, w, dh)
    for name, got, ref, b in zip(("h", "dx", "dw"), (h.detach(), gx, gw), want, bounds):
        assert got.dtype == x.dtype and got.shape == ref.shape
        off = (got.double() - ref).abs()
        assert (off <= b).all(), (name, int((off > b).sum()), float((off / b).max()))
    return h.detach(), gx, gw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,h,f", [(1, 8, 1), (1, 64, 63), (2, 72, 200), (5, 256, 129), (9, 64, 64),
                                   (127, 64, 65), (128, 128, 128), (129, 136, 127), (300, 512, 1365),
                                   (1, 2048, 5632), (2500, 64, 1000), (200, 512, 2001),
                                   (4111, 264, 9001)])
def test_forward_and_gradients(cuda_device, dtype, n, h, f):
    _check(*_data(n, h, f, dtype, n + f, cuda_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,h,f", [
    # few rows, or few blocks of 16 rows: contractions of one batch of loads and just beyond
    (8, 504, 40), (16, 520, 65), (17, 1016, 33), (15, 1032, 31), (9, 2056, 17), (33, 4104, 9),
    (600, 2048, 8), (4700, 8, 3),
    # few rows, more blocks than that: tiles
    (127, 64, 3001), (17, 72, 5000), (100, 520, 2500), (65, 1032, 4800)])
def test_few_rows_and_lone_row_tiles(cuda_device, dtype, n, h, f):
    _check(*_data(n, h, f, dtype, n + f, cuda_device))


@pytest.mark.parametrize("n", [1, 7, 8, 16, 40])
def test_a_row_depends_on_itself_alone(cuda_device, n):
    """Infinities and NaN in one row reach no other; a row alone gives what it gives among others;
    nothing is written beyond the rows and columns of h."""
    from SSA import _lib
    from SSA.ssa_gated_ffn import _problem, ssa_gated_ffn
    x, w, _ = _data(n, 264, 45, torch.bfloat16, 29, cuda_device)
    h = ssa_gated_ffn(x, w)
    bad = x.clone()
    bad[n // 2, 3], bad[n // 2, 200] = float("inf"), float("nan")
    got = ssa_gated_ffn(bad, w)
    other = torch.arange(n, device=cuda_device) != n // 2
    assert torch.equal(got[other], h[other]) and got[n // 2].isnan().all()
    assert torch.equal(ssa_gated_ffn(x[n // 2:n // 2 + 1], w)[0], h[n // 2])
    wide = torch.full((n + 2, 53), 7.0, dtype=x.dtype, device=cuda_device)
    prob = _problem(x, w)
    _lib.check(_lib.load().ssa_gated_ffn_fwd(ctypes.byref(prob), wide[1, 4:].data_ptr(), 53,
                                             _lib.stream_ptr(x.device)))
    assert torch.equal(wide[1:-1, 4:49], h)
    wide[1:-1, 4:49] = 7.0
    assert (wide == 7.0).all()


def test_large_preactivations(cuda_device):
    """Gates of several hundred of both signs: sigmoid 0 and 1, no NaN."""
    _check(*_data(64, 64, 96, torch.bfloat16, 3, cuda_device, scale=100.0))


def test_leading_shape_and_layouts(cuda_device):
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    x, w, dh = _data(60, 64, 90, torch.bfloat16, 5, cuda_device)
    h, gx, gw = _check(x, w, dh)
    assert torch.equal(ssa_gated_ffn(x.view(3, 20, 64), w), h.view(3, 20, 90))
    wide = torch.zeros(60, 80, dtype=x.dtype, device=cuda_device)
    wide[:, 8:72] = x
    odd = torch.zeros(60 * 64 + 1, dtype=x.dtype, device=cuda_device)[1:].view(60, 64)
    odd.copy_(x)
    for xs, ws in ((wide[:, 8:72], w), (odd, w), (x.t().contiguous().t(), w.t().contiguous().t())):
        xl, wl = xs.detach().requires_grad_(True), ws.detach().requires_grad_(True)
        out = ssa_gated_ffn(xl, wl)
        assert torch.equal(out, h)
        for g in (dh, dh.t().contiguous().t(), torch.cat([dh, dh], 1)[:, 90:]):
            a, b = torch.autograd.grad(out, (xl, wl), g, retain_graph=True)
            assert torch.equal(a, gx) and torch.equal(b, gw)
    xl = x.clone().requires_grad_(True)
    (one,) = torch.autograd.grad(ssa_gated_ffn(xl, w).sum(), xl)  # an expanded gradient
    xl2 = x.clone().requires_grad_(True)
    (two,) = torch.autograd.grad(ssa_gated_ffn(xl2, w), xl2, torch.ones_like(h))
    assert torch.equal(one, two)


def test_only_the_asked_gradient_and_empty(cuda_device):
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    x, w, dh = _data(33, 64, 70, torch.bfloat16, 7, cuda_device)
    _, gx, gw = _check(x, w, dh)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ssa_gated_ffn(xl, w), xl, dh)[0], gx)
    assert torch.equal(torch.autograd.grad(ssa_gated_ffn(x, wl), wl, dh)[0], gw)
    e = x[:0].clone().requires_grad_(True)
    out = ssa_gated_ffn(e, wl)
    out.sum().backward()
    assert out.shape == (0, 70) and e.grad.shape == (0, 64) and not wl.grad.any()


def test_gradient_against_differences(cuda_device):
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    x, w, _ = _data(16, 64, 40, torch.float16, 11, cuda_device)
    x, w = (x * 64).round() / 64, (w * 1024).round() / 1024
    g = torch.Generator().manual_seed(13)
    dh = torch.randn(16, 40, generator=g).half().to(cuda_device)
    sx = (torch.randint(0, 2, x.shape, generator=g) * 2 - 1).to(x) / 64
    sw = (torch.randint(0, 2, w.shape, generator=g) * 2 - 1).to(w) / 1024
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(ssa_gated_ffn(xl, wl), (xl, wl), dh)
    f = lambda a, b: float((ssa_gated_ffn(a, b).double() * dh.double()).sum())  # noqa: E731
    slope = float((gx.double() * sx.double()).sum() + (gw.double() * sw.double()).sum())
    X, W = x.double().abs(), w.double().abs()
    move = float((sx.double().abs() @ W.t() + X @ sw.double().abs().t()).max())
    pre = float((x.double() @ w.double().t()).abs().max())
    # |third derivative| of silu(g) u along the direction: silu''' <= 1, silu'' <= 0.5, both moving,
    # and the second-order movement of g and u themselves (sx sw^T)
    cross = float((sx.double().abs() @ sw.double().abs().t()).max())
    third = float(dh.double().abs().sum()) * (move ** 3 * (pre + 1.5) / 6 +
                                              cross * move * (0.5 * pre + 2.2))
    rounding = 2.0 ** -11 * (2 * float((gx.double() * sx.double()).abs().sum()
                                       + (gw.double() * sw.double()).abs().sum())
                             + float((ssa_gated_ffn(x, w).double() * dh.double()).abs().sum()))
    assert abs((f(x + sx, w + sw) - f(x - sx, w - sw)) / 2 - slope) <= third + 2 * rounding


def test_captured_and_replayed(cuda_device):
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    x, w, dh = _data(70, 128, 150, torch.bfloat16, 17, cuda_device)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    def step():
        h = ssa_gated_ffn(xl, wl)
        return h.detach(), *torch.autograd.grad(h, (xl, wl), dh)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    x2, w2, dh2 = _data(70, 128, 150, torch.bfloat16, 18, cuda_device)
    with torch.no_grad():
        xl.copy_(x2)
        wl.copy_(w2)
    dh.copy_(dh2)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, step()):
        assert torch.equal(a, b)


def test_refusals(cuda_device):
    from SSA.ssa_gated_ffn import ssa_gated_ffn as f
    x, w, _ = _data(8, 64, 10, torch.bfloat16, 19, cuda_device)
    for args, match in (((x.float(), w.float()), "fp16 or both bf16"),
                        ((x, w.half()), "fp16 or both bf16"),
                        ((x[:, :60], w[:, :60]), "multiple of 8"), ((x, w[:5]), r"\[2 F, H\]"),
                        ((x, w[:, :32]), r"\[2 F, H\]"), ((x.cpu(), w), "CUDA")):
        with pytest.raises(ValueError, match=match):
            f(*args)


def test_second_derivative_is_refused(cuda_device):
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    x, w, _ = _data(4, 64, 10, torch.bfloat16, 23, cuda_device)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(ssa_gated_ffn(x, w).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
