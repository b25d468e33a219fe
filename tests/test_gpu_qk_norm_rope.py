"""Per-head norm and rotation (SSA.ssa_qk_norm_rope) against the same formulas in 64 bits.

Bounds. All arithmetic is fp32 with one rounding to the output type (u = eps / 2). A forward value is
a few products and one sum: 16 steps of 2^-24 of the magnitudes |n cos| + |rot(n) sin| cover them
(the mean of D <= 128 squares adds D / 16 + 5 more in the norm). The backward has two means and
about twice the products. dw is a sum over rows: the fp32 partial sums of at most 4096 terms per
thread are off by 4096 2^-24 of the sum of magnitudes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _tables(rows, d, dev):
    import luciole_train as LT
    return LT.rope_tables(rows, d, 10000.0, dev)


def _rot(x):
    a, b = x.chunk(2, -1)
    return torch.cat([-b, a], -1)


def _reference(qkv, hq, hkv, cos, sin, wq, wk, eps, at):
    """q, k, v in fp64 (differentiable) and the magnitudes that bound the forward's error."""
    d = cos.shape[1]
    x = qkv.unflatten(-1, (hq + 2 * hkv, d))
    q, k, v = x.split([hq, hkv, hkv], -2)
    c, s = cos.double()[at].unsqueeze(-2), sin.double()[at].unsqueeze(-2)

    def one(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w
        return y * c + _rot(y) * s, (y * c).abs() + (_rot(y) * s).abs()

    (q, mq), (k, mk) = one(q, wq), one(k, wk)
    return (q, k, v), (mq.detach(), mk.detach())


def _check(lead, hq, hkv, d, dtype, dev, norm, positions=None, rows=None, seed=0, w_dtype=None,
           layout=lambda t: t):
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    g = torch.Generator().manual_seed(seed)
    eps = 1e-5
    qkv = layout(torch.randn(*lead, (hq + 2 * hkv) * d, generator=g).to(dtype).to(dev))
    cos, sin = _tables(rows or lead[-1], d, dev)
    ws = [(1 + 0.2 * torch.randn(d, generator=g)).to(w_dtype or dtype).to(dev) if norm else None
          for _ in range(2)]
    grads = [torch.randn(*lead, h, d, generator=g).to(dtype).to(dev) for h in (hq, hkv, hkv)]
    at = positions if positions is not None else torch.arange(lead[-1], device=dev)
    leaves = [qkv.detach().requires_grad_(True)] + [w.requires_grad_(True) for w in ws if norm]
    out = ssa_qk_norm_rope(leaves[0], hq, hkv, cos, sin, *(ws if norm else (None, None)), eps=eps,
                           positions=positions)
    got = torch.autograd.grad(out, leaves, grads)
    ref_leaves = [t.detach().double().requires_grad_(True) for t in leaves]
    want, mags = _reference(ref_leaves[0], hq, hkv, cos, sin, *(ref_leaves[1:] if norm else (None, None)),
                            eps, at.long())
    ref = torch.autograd.grad(want, ref_leaves, [t.double() for t in grads])
    u, e = torch.finfo(dtype).eps / 2, 2.0 ** -24
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    steps = 16 + (d / 16 + 5 if norm else 0)
    for name, o, r, m in (("q", out[0], want[0], mags[0]), ("k", out[1], want[1], mags[1])):
        assert o.shape == r.shape and o.dtype == dtype
        off = (o.double() - r).detach().abs()
        assert (off <= u * r.detach().abs() + steps * e * m + tiny).all(), (name, float(off.max()))
    assert torch.equal(out[2], qkv.unflatten(-1, (hq + 2 * hkv, d))[..., hq + hkv:, :])
    # |dqkv| terms: |dn| <= |dy cos| + |dy sin|, times w r, plus the projection of at most its size
    x = qkv.double().unflatten(-1, (hq + 2 * hkv, d))
    dy = torch.cat([t.double() for t in grads], -2)
    mag = dy.abs() + _rot(dy).abs()
    scale = torch.ones_like(mag[..., :1])
    if norm:
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
        w = torch.cat([ws[0].double().abs().expand(hq, d), ws[1].double().abs().expand(hkv, d),
                       torch.ones(hkv, d, device=dev)]).detach()
        mag = mag * w
        mag = mag + (x * r).abs() * (mag * (x * r).abs()).mean(-1, keepdim=True)
        scale = r
    bound = u * ref[0].abs() + 2 * steps * e * (mag * scale).flatten(-2) + tiny
    off = (got[0].double() - ref[0]).abs()
    assert got[0].dtype == dtype and (off <= bound).all(), ("dqkv", float((off / bound).max()))
    if norm:
        full = (dy.abs() + _rot(dy).abs()) * (x * r).abs()
        for i, (lo, hi) in enumerate(((0, hq), (hq, hq + hkv))):
            uw = torch.finfo(ws[i].dtype).eps / 2
            b = uw * ref[1 + i].abs() + 4096 * e * full[..., lo:hi, :].reshape(-1, d).sum(0)
            assert got[1 + i].dtype == ws[i].dtype
            assert ((got[1 + i].double() - ref[1 + i]).abs() <= b).all(), ("dw", i)
    return [t.detach() for t in out] + list(got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("lead,hq,hkv,d", [((1, 1), 1, 1, 16), ((3,), 5, 1, 128), ((2, 77), 6, 2, 32),
                                           ((1000,), 24, 8, 64), ((2, 1500), 32, 8, 64),
                                           ((700,), 32, 8, 128), ((9000,), 15, 5, 16)])
def test_forward_and_gradients(cuda_device, dtype, norm, lead, hq, hkv, d):
    _check(lead, hq, hkv, d, dtype, cuda_device, norm, seed=hq + d)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions(cuda_device, kind):
    dev = cuda_device
    g = torch.Generator().manual_seed(3)
    for shape, lead in (((50,), (50,)), ((40,), (3, 40)), ((3, 40), (3, 40))):
        pos = torch.randint(0, 130000, shape, generator=g).to(kind).to(dev)
        _check(lead, 4, 2, 64, torch.bfloat16, dev, True, positions=pos, rows=130000)
    # every row at one position
    _check((33,), 4, 2, 64, torch.float32, dev, True,
           positions=torch.full((33,), 129999, dtype=kind, device=dev), rows=130000)


def test_position_outside_the_tables_is_nan(cuda_device):
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    dev = cuda_device
    cos, sin = _tables(16, 32, dev)
    qkv = torch.randn(5, 4 * 32, device=dev, dtype=torch.bfloat16, requires_grad=True)
    pos = torch.tensor([0, 16, 15, -1, 2 ** 40], device=dev)
    q, k, v = ssa_qk_norm_rope(qkv, 2, 1, cos, sin, positions=pos)
    assert torch.isnan(q).all((1, 2)).tolist() == [False, True, False, True, True]
    assert torch.isnan(k).any((1, 2)).tolist() == [False, True, False, True, True]
    assert not torch.isnan(v).any()


def test_fp32_weights_and_layouts(cuda_device):
    dev = cuda_device
    base = _check((2, 31), 4, 2, 64, torch.bfloat16, dev, True, seed=7)
    _check((2, 31), 4, 2, 64, torch.bfloat16, dev, True, seed=7, w_dtype=torch.float32)

    def wide(t):
        o = torch.zeros(*t.shape[:-1], t.shape[-1] + 24, dtype=t.dtype, device=dev)
        o[..., 8:-16] = t
        return o[..., 8:-16]

    def odd(t):
        o = torch.zeros(t.numel() + 3, dtype=t.dtype, device=dev)[3:].view(t.shape)
        return o.copy_(t)

    def swapped(t):  # sequence-major storage, as Megatron keeps it
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    for layout in (wide, odd, swapped):
        for a, b in zip(base, _check((2, 31), 4, 2, 64, torch.bfloat16, dev, True, seed=7,
                                     layout=layout)):
            assert torch.equal(a, b)


def test_gradients_in_attention_layout_and_missing_ones(cuda_device):
    """dq and dk as [B, H, S, D] storage seen as [B, S, H, D]; an output that is not used."""
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    dev = cuda_device
    g = torch.Generator().manual_seed(5)
    cos, sin = _tables(40, 64, dev)
    qkv = torch.randn(2, 40, 8 * 64, generator=g).bfloat16().to(dev).requires_grad_(True)
    q, k, v = ssa_qk_norm_rope(qkv, 4, 2, cos, sin)
    dq, dk, dv = (torch.randn(t.shape, generator=g).bfloat16().to(dev) for t in (q, k, v))
    (want,) = torch.autograd.grad((q, k, v), qkv, (dq, dk, dv), retain_graph=True)
    hm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (dq, dk, dv)]
    (got,) = torch.autograd.grad((q, k, v), qkv, hm, retain_graph=True)
    assert torch.equal(got, want)
    (only,) = torch.autograd.grad(q, qkv, dq)
    assert torch.equal(only[..., :256], want[..., :256]) and not only[..., 256:].any()


def test_same_as_the_decoders_rotation(cuda_device):
    import luciole_train as LT
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    dev = cuda_device
    qkv = torch.randn(2, 300, 12 * 64, device=dev)
    cos, sin = _tables(300, 64, dev)
    q, k, v = ssa_qk_norm_rope(qkv, 8, 2, cos, sin)
    x = qkv.view(2, 300, 12, 64)
    # fp32: three roundings each
    assert (q - LT.apply_rope(x[:, :, :8], cos, sin)).abs().max() <= 4 * 2.0 ** -23 * x.abs().max()
    assert (k - LT.apply_rope(x[:, :, 8:10], cos, sin)).abs().max() <= 4 * 2.0 ** -23 * x.abs().max()


def test_empty(cuda_device):
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    cos, sin = _tables(4, 32, cuda_device)
    qkv = torch.zeros(0, 4 * 32, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(32, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    q, k, v = ssa_qk_norm_rope(qkv, 2, 1, cos, sin, w, w)
    assert q.shape == (0, 2, 32) and k.shape == (0, 1, 32) and v.shape == (0, 1, 32)
    (q.sum() + k.sum()).backward()
    assert not w.grad.any()


def test_captured_and_replayed(cuda_device):
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    dev = cuda_device
    cos, sin = _tables(64, 64, dev)
    qkv = torch.randn(2, 64, 8 * 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    w = [torch.ones(64, device=dev, dtype=torch.bfloat16, requires_grad=True) for _ in range(2)]
    gs = [torch.randn(2, 64, h, 64, device=dev, dtype=torch.bfloat16) for h in (4, 2, 2)]

    def step():
        out = ssa_qk_norm_rope(qkv, 4, 2, cos, sin, *w)
        return [t.detach().clone() for t in out] + list(torch.autograd.grad(out, [qkv] + w, gs))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.no_grad():
        qkv.copy_(torch.randn(2, 64, 8 * 64, device=dev))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, step()):
        assert torch.equal(a, b)


def test_refusals(cuda_device):
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope as f
    dev = cuda_device
    cos, sin = _tables(8, 64, dev)
    x = torch.zeros(2, 8, 8 * 64, device=dev, dtype=torch.bfloat16)
    w = torch.ones(64, device=dev, dtype=torch.bfloat16)
    pos = torch.zeros(8, dtype=torch.int32, device=dev)
    for args, kw, match in (
            ((x[..., :-64], 4, 2, cos, sin), {}, "must be"),
            ((x, 0, 4, cos, sin), {}, "must be"),
            ((x, 4, 2, cos.double(), sin.double()), {}, "fp32"),
            ((x, 4, 2, cos[:, :48], sin[:, :48]), {}, "head dim"),
            ((x, 4, 2, cos[:7], sin[:7]), {}, "7 positions"),
            ((x, 4, 2, cos, sin, w), {}, "together"),
            ((x, 4, 2, cos, sin, w[:32], w[:32]), {}, r"\[64\]"),
            ((x, 4, 2, cos, sin, w.half(), w.half()), {}, r"\[64\]"),
            ((x, 4, 2, cos, sin), {"positions": pos[:4]}, "positions"),
            ((x, 4, 2, cos, sin), {"positions": pos.float()}, "int32 or int64"),
            ((x.cpu(), 4, 2, cos, sin), {}, "CUDA"),
            ((x.double(), 4, 2, cos, sin), {}, "dtype")):
        with pytest.raises(ValueError, match=match):
            f(*args, **kw)
