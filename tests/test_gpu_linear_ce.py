"""Linear cross entropy (SSA.ssa_cross_entropy) against the same formulas in 64 bits.

Bounds. A logit is a sum of H exact products of 16-bit values in fp32 accumulators: H / 16 matrix
instructions, each adding with an error of at most a few steps of 2^-23 relative to the sum of
magnitudes A = sum |x||w|; DL = (H / 8 + 8) 2^-23 A bounds it. A row's loss is off by at most
2 DL plus a few fp32 roundings of the loss. d is rounded once to 16 bits (u = eps / 2 relative) after
exponentials whose argument is off by up to 2 DL, the sums over it run in fp32, and the result is
rounded once: |dx error| <= (u + 2 DL + 2^-16) |d| |W| + u |dx|, elementwise. With one gradient per
row (reduction "none") its fraction multiplies x in the sum for dW and that product is rounded to 16
bits as well: each term is a product of two rounded factors, so dW's bound has 2 u (and u^2, inside
2^-16) where the others have u."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _data(n, h, v, dtype, seed, ignored, dev, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, h, generator=g).to(dtype).to(dev)
    w = (torch.randn(v, h, generator=g) * (scale / math.sqrt(h))).to(dtype).to(dev)
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.rand(n, generator=g) < ignored] = -100
    return x, w, t.to(dev)


def _reference(x, w, t, reduction, grad, ignore_index=-100):
    """loss, dx, dW in fp64, and the elementwise bounds of the module docstring."""
    X, W = x.double(), w.double()
    logits = X @ W.t()
    lse = torch.logsumexp(logits, 1)
    keep = t != ignore_index
    at = torch.where(keep, t, torch.zeros_like(t)).long()
    rows = torch.where(keep, lse - logits.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    n = keep.sum()
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / n}[reduction]
    gr = torch.where(keep, grad.double() * torch.ones_like(rows) / (n if reduction == "mean" else 1),
                     torch.zeros_like(rows))
    d = torch.exp(logits - lse[:, None])
    d[torch.arange(len(t), device=t.device), at] -= 1.0
    d = d * gr[:, None]
    u = torch.finfo(x.dtype).eps / 2
    dl = (x.shape[1] / 8 + 8) * 2.0 ** -23 * float((X.abs() @ W.abs().t()).max())
    e = u + 2 * dl + 2.0 ** -16
    dx, dw = d @ W, d.t() @ X
    # the target's d = p - 1 carries p's error: |p| <= |d| + 1 there; fp16 d below its normal range
    # is off by 2^-25 of the scale 2^-11 max |g|; an exponential below 2^-126, the smallest normal
    # fp32 number, is flushed to zero (logits of several hundred reach that)
    slack = gr.abs().max() * 2.0 ** (-36 if x.dtype == torch.float16 else -126)
    D = d.abs() + slack
    D[torch.arange(len(t), device=t.device), at] += 2 * dl * gr.abs()
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps  # subnormal results: half a step
    bdx = e * (D @ W.abs()) + u * dx.abs() + tiny
    bdw = (e + (u if reduction == "none" else 0.0)) * (D.t() @ X.abs()) + u * dw.abs() + tiny
    return loss, dx, dw, 2 * dl, bdx, bdw


def _check(x, w, t, reduction="mean", grad=None, ignore_index=-100):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = ssa_linear_cross_entropy(xl, wl, t, ignore_index=ignore_index, reduction=reduction)
    if grad is None:
        grad = torch.rand(loss.shape, device=x.device) + 0.5
    gx, gw = torch.autograd.grad(loss, (xl, wl), grad)
    ref, dx, dw, bl, bdx, bdw = _reference(x, w, t, reduction, grad, ignore_index)
    assert loss.dtype == torch.float32 and gx.dtype == x.dtype and gw.shape == w.shape
    n = max(1, int((t != ignore_index).sum()))
    bound = bl * (n if reduction == "sum" else 1) + 2.0 ** -20 * (ref.abs() + 1)
    assert ((loss.double() - ref).abs() <= bound).all(), (loss, ref)
    for name, got, want, b in (("dx", gx, dx, bdx), ("dw", gw, dw, bdw)):
        bad = ((got.double() - want).abs() > b)
        assert not bad.any(), (name, int(bad.sum()), float(((got.double() - want).abs() / b).max()))
    return loss, gx, gw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,h,v", [(1, 8, 1), (1, 64, 1000), (3, 72, 257), (127, 64, 255),
                                   (128, 128, 256), (129, 136, 1021), (300, 512, 3001),
                                   (640, 256, 8191), (1, 2048, 50257), (257, 64, 70001)])
def test_loss_and_gradients(cuda_device, dtype, n, h, v):
    x, w, t = _data(n, h, v, dtype, n + v, 0.2 if n > 1 else 0.0, cuda_device)
    t[0] = v - 1
    _check(x, w, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,h,v", [
    # few rows, or few steps of 16 rows: contractions of one batch of loads and beyond, blocks of one
    # step and of several
    (2, 520, 300), (8, 1032, 1000), (9, 64, 33), (16, 1024, 4000), (17, 2056, 700), (60, 264, 500),
    (300, 512, 16), (5, 64, 20001), (8, 1032, 10007), (16, 1032, 9000),
    # few rows, more steps than that: tiles
    (17, 72, 20000), (100, 520, 20001), (9, 2056, 10000)])
def test_few_rows_and_lone_row_tiles(cuda_device, dtype, n, h, v):
    _check(*_data(n, h, v, dtype, n + v, 0.2 if n > 2 else 0.0, cuda_device))


@pytest.mark.parametrize("n", [3, 8, 11, 40])
def test_a_row_depends_on_itself_alone(cuda_device, n):
    """Infinities and NaN in one row reach no other row's loss, and every target of the vocabulary's
    ends and steps is found."""
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(n, 264, 1003, torch.bfloat16, 31, 0.0, cuda_device)
    ends = torch.tensor([0, 1002, 15, 16, 31, 32, 1000, 991, 7, 8], device=cuda_device)
    t[:min(n, 10)] = ends[:n]
    loss = ssa_linear_cross_entropy(x, w, t, reduction="none")
    logits = x.double() @ w.double().t()
    want = torch.logsumexp(logits, 1) - logits.gather(1, t[:, None])[:, 0]
    dl = (264 / 8 + 8) * 2.0 ** -23 * float((x.double().abs() @ w.double().abs().t()).max())
    assert ((loss.double() - want).abs() <= 2 * dl + 2.0 ** -20 * (want.abs() + 1)).all()
    bad = x.clone()
    bad[n // 2, 3], bad[n // 2, 200] = float("inf"), float("nan")
    got = ssa_linear_cross_entropy(bad, w, t, reduction="none")
    other = torch.arange(n, device=cuda_device) != n // 2
    assert torch.equal(got[other], loss[other]) and got[n // 2].isnan()


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions_and_leading_shape(cuda_device, reduction):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(200, 128, 777, torch.bfloat16, 5, 0.3, cuda_device)
    loss, _, _ = _check(x, w, t, reduction)
    again = ssa_linear_cross_entropy(x.view(4, 50, 128), w, t.view(4, 50).int(), reduction=reduction)
    assert again.shape == ((4, 50) if reduction == "none" else ())
    assert torch.equal(again.reshape(-1), loss.detach().reshape(-1))


def test_many_pieces_equal_one(cuda_device):
    """Enough rows that the vocabulary is walked in several pieces (20,000 rows: 6,656 columns)."""
    x, w, t = _data(20000, 64, 20011, torch.bfloat16, 9, 0.1, cuda_device)
    _check(x, w, t)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_long_contractions(cuda_device, reduction):
    """Sizes at which dx and dW take the 256 x 512 tiles, none of them a multiple of a tile."""
    x, w, t = _data(4300, 520, 16001, torch.bfloat16, 15, 0.1, cuda_device)
    _check(x, w, t, reduction)


def test_row_weights_of_widely_different_size(cuda_device):
    x, w, t = _data(96, 128, 999, torch.float16, 11, 0.1, cuda_device)
    grad = torch.logspace(-3, 3, 96, device=cuda_device)
    _check(x, w, t, "none", grad)
    _check(x, w, t, "none", torch.zeros(96, device=cuda_device))


def test_ignored_rows_and_ids(cuda_device):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(64, 64, 100, torch.bfloat16, 13, 0.0, cuda_device)
    t[::2] = 7
    _check(x, w, t, ignore_index=7)                  # an id of the vocabulary
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    none = torch.full_like(t, -100)
    loss = ssa_linear_cross_entropy(xl, wl, none)
    gx, gw = torch.autograd.grad(loss, (xl, wl))
    assert torch.isnan(loss) and not gx.any() and not gw.any()
    assert float(ssa_linear_cross_entropy(x, w, none, reduction="sum")) == 0.0
    bad = t.clone()
    bad[3], bad[5] = 100, -1                          # out of range: NaN, nothing read
    rows = ssa_linear_cross_entropy(x, w, bad, reduction="none")
    assert torch.isnan(rows).nonzero()[:, 0].tolist() == [3, 5]
    # all rows with one target: its gradient row sums over every row
    _check(x, w, torch.full_like(t, 99))


def test_large_logits(cuda_device):
    """Logits of several hundred: the loss does not lose the difference."""
    x, w, t = _data(130, 256, 600, torch.bfloat16, 17, 0.0, cuda_device, scale=200.0)
    _check(x, w, t, "none")


def test_layouts(cuda_device):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(70, 64, 301, torch.bfloat16, 19, 0.1, cuda_device)
    want = _check(x, w, t, "none", torch.ones(70, device=cuda_device))[0]
    wide = torch.zeros(70, 80, dtype=x.dtype, device=cuda_device)
    wide[:, 8:72] = x
    odd = torch.zeros(70 * 64 + 1, dtype=x.dtype, device=cuda_device)[1:].view(70, 64)
    odd.copy_(x)
    for xs, ws in ((wide[:, 8:72], w), (odd, w), (x.t().contiguous().t(), w.t().contiguous().t())):
        assert torch.equal(ssa_linear_cross_entropy(xs, ws, t, reduction="none"), want)
    one = x[:1].expand(70, 64)
    same = ssa_linear_cross_entropy(one, w, torch.zeros_like(t), reduction="none")
    assert (same == same[0]).all()


def test_empty_batch(cuda_device):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(4, 64, 50, torch.bfloat16, 21, 0.0, cuda_device)
    xl, wl = x[:0].clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = ssa_linear_cross_entropy(xl, wl, t[:0], reduction="sum")
    loss.backward()
    assert float(loss.detach()) == 0.0 and xl.grad.shape == (0, 64) and not wl.grad.any()


def test_only_the_asked_gradient(cuda_device):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(90, 64, 500, torch.bfloat16, 23, 0.1, cuda_device)
    _, gx, gw = _check(x, w, t, "sum", torch.ones((), device=cuda_device))
    xl = x.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(
        ssa_linear_cross_entropy(xl, w, t, reduction="sum"), xl)[0], gx)
    wl = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(
        ssa_linear_cross_entropy(x, wl, t, reduction="sum"), wl)[0], gw)


def test_gradient_against_differences(cuda_device):
    """Central differences of the fp32 loss along a direction of both inputs: steps of fp16-exact
    size keep x +- s and w +- s exact."""
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(64, 64, 211, torch.float16, 29, 0.1, cuda_device, scale=1.0)
    x, w = (x * 64).round() / 64, (w * 1024).round() / 1024
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = ssa_linear_cross_entropy(xl, wl, t, reduction="sum")
    gx, gw = torch.autograd.grad(loss, (xl, wl))
    g = torch.Generator().manual_seed(31)
    sx = (torch.randint(0, 2, x.shape, generator=g) * 2 - 1).to(x) / 64
    sw = (torch.randint(0, 2, w.shape, generator=g) * 2 - 1).to(w) / 1024
    up = ssa_linear_cross_entropy(x + sx, w + sw, t, reduction="none").double().sum()
    dn = ssa_linear_cross_entropy(x - sx, w - sw, t, reduction="none").double().sum()
    slope = float((gx.double() * sx.double()).sum() + (gw.double() * sw.double()).sum())
    # the third-order term: a logit moves by at most |sx||w| + |x||sw| along the direction
    move = float((sx.double().abs() @ w.double().abs().t()
                  + x.double().abs() @ sw.double().abs().t()).max())
    third = 64 * move ** 3 / 3
    rounding = 2.0 ** -11 * 2 * float((gx.double() * sx.double()).abs().sum()
                                      + (gw.double() * sw.double()).abs().sum())
    assert abs(float(up - dn) / 2 - slope) <= third + rounding + 1e-3


def test_captured_and_replayed(cuda_device):
    """Forward and backward in one CUDA graph, replayed on new inputs, on a stream of their own."""
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w, t = _data(150, 128, 1234, torch.bfloat16, 37, 0.1, cuda_device)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    def step():
        loss = ssa_linear_cross_entropy(xl, wl, t)
        return loss.detach(), *torch.autograd.grad(loss, (xl, wl))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    x2, w2, t2 = _data(150, 128, 1234, torch.bfloat16, 38, 0.5, cuda_device)
    with torch.no_grad():
        xl.copy_(x2)
        wl.copy_(w2)
    t.copy_(t2)
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)


def test_refusals(cuda_device):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy as f
    x, w, t = _data(8, 64, 50, torch.bfloat16, 41, 0.0, cuda_device)
    for args, kw, match in (
            ((x.float(), w.float(), t), {}, "fp16 or both bf16"),
            ((x, w.half(), t), {}, "fp16 or both bf16"),
            ((x[:, :60], w[:, :60], t), {}, "multiple of 8"),
            ((x, w[:, :32], t), {}, "shape mismatch"),
            ((x, w, t[:4]), {}, "leading shape"),
            ((x, w, t.float()), {}, "int64 or int32"),
            ((x, w, t), {"reduction": "max"}, "reduction"),
            ((x.cpu(), w, t), {}, "CUDA")):
        with pytest.raises(ValueError, match=match):
            f(*args, **kw)


def test_what_an_ignored_row_holds_reaches_nothing(cuda_device):
    """Infinities and NaN in the hidden states of ignored rows (padding): the other rows' losses and
    every gradient are as without them."""
    x, w, t = _data(200, 128, 777, torch.bfloat16, 43, 0.3, cuda_device)
    want = _check(x, w, t)
    dirty = x.clone()
    skip = t == -100
    dirty[skip] = float("nan")
    dirty[skip.nonzero()[0, 0]] = float("inf")
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    xl, wl = dirty.requires_grad_(True), w.clone().requires_grad_(True)
    loss = ssa_linear_cross_entropy(xl, wl, t)
    assert torch.equal(loss, want[0])
    grad = torch.rand(loss.shape, device=x.device) + 0.5
    gx, gw = torch.autograd.grad(loss, (xl, wl), grad)
    clean = x.clone().requires_grad_(True)
    a, b = torch.autograd.grad(ssa_linear_cross_entropy(clean, wl, t), (clean, wl), grad)
    assert torch.equal(gx, a) and torch.equal(gw, b) and not gx[skip].any()


def test_two_streams_at_once(cuda_device):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    sets = [_data(700, 256, 9001, torch.bfloat16, 50 + i, 0.1, cuda_device) for i in range(2)]

    def step(x, w, t):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = ssa_linear_cross_entropy(x, w, t)
        return [loss.detach(), *torch.autograd.grad(loss, (x, w))]

    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i] = step(*s)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_device_timeout_shows_as_nan(cuda_device):
    """With the device status set (a self-test wait that runs out), the tensor-core products write NaN;
    once it is read, results are back."""
    from SSA import _lib, check_device_status
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    x, w, t = _data(300, 128, 2000, torch.bfloat16, 61, 0.1, cuda_device)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    good = ssa_linear_cross_entropy(xl, wl, t)
    fw = w[:1000].detach()
    h = ssa_gated_ffn(x, fw)
    lib = _lib.load()
    _lib.check(lib.ssa_selftest_device_timeout(1_000_000, _lib.stream_ptr(cuda_device)))
    bad = ssa_linear_cross_entropy(xl, wl, t)
    gx, gw = torch.autograd.grad(good, (xl, wl), retain_graph=True)
    assert torch.isnan(bad) and torch.isnan(gx[t != -100]).all() and torch.isnan(gw).all()
    assert torch.isnan(ssa_gated_ffn(x, fw)).all()
    with pytest.raises(_lib.SSAKernelError):
        check_device_status()
    assert torch.equal(ssa_linear_cross_entropy(xl, wl, t), good)
    assert torch.equal(ssa_gated_ffn(x, fw), h)
