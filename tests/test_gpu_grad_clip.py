"""Global gradient norm and clipping (SSA.ssa_grad_clip) against the same sums in 64 bits.

Bounds. A thread adds at most 32 squares in fp32 (33 steps of 2^-24), everything above that in fp64,
and the norm is rounded once: 20 steps of 2^-24 relative after the square root. An element is multiplied in
fp32 by a coefficient off by that and three more roundings, and rounded once to its type."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

REL = 20 * 2.0 ** -24


def _grads(sizes, dtype, dev, seed=0, scale=0.1):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtype).to(dev) for s in sizes]


def _norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def _check(grads, max_norm, out=None):
    from SSA.ssa_grad_clip import ssa_clip_grad_norm, ssa_grad_norm
    norm = _norm64(grads)
    before = [g.double() for g in grads]
    assert abs(float(ssa_grad_norm(grads)) - norm) <= REL * norm
    got = ssa_clip_grad_norm(grads, max_norm, out=out)
    assert got.dtype == torch.float32 and abs(float(got) - norm) <= REL * norm
    coef = min(1.0, max_norm / (norm + 1e-6))
    for b, g, o in zip(before, grads, out if out is not None else grads):
        u = torch.finfo(o.dtype).eps / 2
        want = b * coef
        tiny = torch.finfo(o.dtype).tiny * torch.finfo(o.dtype).eps
        assert ((o.double() - want).abs() <= (u + REL + 2.0 ** -22) * want.abs() + tiny).all()
        if out is not None:
            assert torch.equal(g.double(), b)
        elif coef == 1.0:
            assert torch.equal(o.double(), b)


SIZES = [[(1,)], [(7,), (0,), (3, 5)], [(16384,), (16385,), (16383,), (1,), (2, 100003)],
         [(33,)] * 65, [(5, 1 + i % 7) for i in range(1600)]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", SIZES, ids=["one", "empty", "chunks", "65", "1600"])
@pytest.mark.parametrize("clipped", [True, False])
def test_in_place_and_into(cuda_device, dtype, sizes, clipped):
    dev = cuda_device
    max_norm = 0.05 if clipped else 1e6
    _check(_grads(sizes, dtype, dev), max_norm)
    for o in {torch.float32, dtype}:
        out = [torch.full(s, 7.0, dtype=o, device=dev) for s in sizes]
        _check(_grads(sizes, dtype, dev), max_norm, out)


def test_matches_torch(cuda_device):
    from SSA.ssa_grad_clip import ssa_clip_grad_norm
    ps = [torch.nn.Parameter(torch.zeros(n, device=cuda_device)) for n in (1000, 77, 50000)]
    for p in ps:
        p.grad = torch.randn_like(p)
    mine = [p.grad.clone() for p in ps]
    total = torch.nn.utils.clip_grad_norm_(ps, 1.5)
    norm = ssa_clip_grad_norm(mine, 1.5)
    assert abs(float(norm) - float(total)) <= 1e-5 * float(total)  # torch sums in fp32
    for p, m in zip(ps, mine):
        assert torch.allclose(p.grad, m, rtol=2e-5, atol=0)


def test_the_factor_is_rounded_once(cuda_device):
    """max_norm and the norm's root stay in 64 bits up to the factor: all elements carry its one
    rounding, 2^-24 at most, and the norm's squares here are exact (a power of two times integers)."""
    from SSA.ssa_grad_clip import ssa_clip_grad_norm
    g = torch.full((4096,), 0.5, device=cuda_device)  # norm 32
    for max_norm in (0.1, 0.3, 1.7, 3.3, 1 / 3, 31.9):
        out = torch.empty_like(g)
        assert float(ssa_clip_grad_norm([g], max_norm, out=[out])) == 32.0
        want = max_norm / (32.0 + 1e-6)
        assert abs(float(out[0]) / 0.5 - want) <= 2.0 ** -24 * want and (out == out[0]).all()


def test_range_of_squares(cuda_device):
    """Squares that overflow or underflow fp32."""
    from SSA.ssa_grad_clip import ssa_grad_norm
    for scale in (1e30, 1e-30, 1e-20, 1e18):
        g = _grads([(5000,), (20000,)], torch.float32, cuda_device, 3, scale)
        norm = _norm64(g)
        assert abs(float(ssa_grad_norm(g)) - norm) <= REL * norm
    mixed = _grads([(100,)], torch.float32, cuda_device, 4, 1e25) + \
        _grads([(100,)], torch.float32, cuda_device, 5, 1e-25)
    assert abs(float(ssa_grad_norm(mixed)) - _norm64(mixed)) <= REL * _norm64(mixed)
    assert float(ssa_grad_norm([torch.zeros(70000, device=cuda_device)])) == 0.0


def test_infinities_and_nan_as_torch(cuda_device):
    from SSA.ssa_grad_clip import ssa_clip_grad_norm
    for bad in (float("inf"), float("nan")):
        ps = [torch.nn.Parameter(torch.zeros(100, device=cuda_device)) for _ in range(2)]
        for p in ps:
            p.grad = torch.ones_like(p)
        ps[0].grad[3] = bad
        mine = [p.grad.clone() for p in ps]
        total = torch.nn.utils.clip_grad_norm_(ps, 1.0)
        norm = ssa_clip_grad_norm(mine, 1.0)
        assert torch.equal(norm.isnan(), total.isnan()) and torch.equal(norm.isinf(), total.isinf())
        for p, m in zip(ps, mine):
            assert torch.equal(p.grad.isnan(), m.isnan())
            assert torch.equal(p.grad.nan_to_num(), m.nan_to_num())


def test_layouts(cuda_device):
    """Views that start off a 16-byte boundary, and gradients that are not contiguous."""
    dev = cuda_device
    flat = _grads([(50007,)], torch.bfloat16, dev)[0]
    _check([flat[1:30000], flat[30000:30003], flat[30003:]], 0.01)
    a = _grads([(300, 200)], torch.float32, dev)[0]
    _check([a.t(), _grads([(64, 32)], torch.float32, dev)[0][:, ::2]], 0.01)
    out = torch.zeros(10001, device=dev)
    _check([flat[1:10001].float()], 0.01, [out[1:]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("start", [0, 1, 8])
def test_ends_of_tensors(cuda_device, dtype, start):
    """Sizes around the vectors, the batches and the 64 KB chunks the kernels walk in, from aligned and
    unaligned starts; what lies before and behind a tensor stays as it was."""
    chunk = 65536 // torch.finfo(dtype).bits * 8
    sizes = [1, 3, 4, 5, 7, 8, 9, 2047, 2049, 4099, chunk - 9, chunk - 8, chunk - 1, chunk + 1,
             chunk + 8, chunk + 2051, 2 * chunk - 3]
    flats = _grads([(start + n + 16,) for n in sizes], dtype, cuda_device, seed=start + 1)
    views = [f[start:start + n] for f, n in zip(flats, sizes)]
    whole = [f.clone() for f in flats]
    for o in {torch.float32, dtype}:
        outs = [torch.full((start + n + 16,), 7.0, dtype=o, device=cuda_device) for n in sizes]
        _check(views, 0.05, [t[start:start + n] for t, n in zip(outs, sizes)])
        for t, n in zip(outs, sizes):
            assert (t[:start] == 7.0).all() and (t[start + n:] == 7.0).all()
    _check(views, 0.05)
    for f, w, n in zip(flats, whole, sizes):
        assert torch.equal(f[:start], w[:start]) and torch.equal(f[start + n:], w[start + n:])


def test_repeatable_and_captured(cuda_device):
    from SSA.ssa_grad_clip import ssa_clip_grad_norm
    grads = _grads([(100000,), (3, 7), (511,)], torch.bfloat16, cuda_device)
    out = [torch.zeros(g.shape, device=cuda_device) for g in grads]
    n1 = ssa_clip_grad_norm(grads, 0.3, out)
    first = [o.clone() for o in out]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n2 = ssa_clip_grad_norm(grads, 0.3, out)
    for o in out:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(n1, n2) and all(torch.equal(a, b) for a, b in zip(first, out))
    new = _grads([(100000,), (3, 7), (511,)], torch.bfloat16, cuda_device, 9)
    for g, n in zip(grads, new):
        g.copy_(n)
    graph.replay()
    torch.cuda.synchronize()
    want = [torch.zeros_like(o) for o in out]
    assert torch.equal(ssa_clip_grad_norm(new, 0.3, want), n2)
    assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_in_place_is_seen_by_autograd(cuda_device):
    from SSA.ssa_grad_clip import ssa_clip_grad_norm
    g = torch.ones(8, device=cuda_device)
    v = g._version
    ssa_clip_grad_norm([g], 1.0)
    assert g._version > v


def test_refusals(cuda_device):
    from SSA.ssa_grad_clip import ssa_clip_grad_norm, ssa_grad_norm
    dev = cuda_device
    a, b = torch.ones(8, device=dev), torch.ones(8, device=dev)
    assert float(ssa_clip_grad_norm([], 1.0)) == 0.0 and float(ssa_grad_norm([])) == 0.0
    for grads, kw, match in (
            ([a, b.half()], {}, "one dtype"), ([a.cpu()], {}, "CUDA"),
            ([a.double()], {}, "fp32, fp16 or bf16"), ([a, 1.0], {}, "dense"),
            ([a, a], {}, "share memory"), ([a, a[4:]], {}, "share memory"),
            ([a.expand(3, 8)], {}, "share memory"),
            ([a, b], {"out": [a]}, "2 gradients"), ([a], {"out": [b[:4]]}, "shape"),
            ([a], {"out": [b.half()]}, "fp32 or"), ([a.half()], {"out": [b.bfloat16()]}, "fp32 or"),
            ([a, b], {"out": [b, a]}, "share memory"),
            ([a[:4].half()], {"out": [torch.ones(8, device=dev)[::2]]}, "contiguous"),
            ([a], {"max_norm": -1.0}, "max_norm"), ([a], {"max_norm": float("nan")}, "max_norm")):
        kw = dict({"max_norm": 1.0}, **kw)
        with pytest.raises(ValueError, match=match):
            ssa_clip_grad_norm(grads, **kw)
    assert torch.equal(a, torch.ones(8, device=dev))


def test_only_empty_tensors(cuda_device):
    from SSA.ssa_grad_clip import ssa_clip_grad_norm, ssa_grad_norm
    empty = [torch.zeros(0, 3, device=cuda_device), torch.zeros(0, device=cuda_device)]
    assert float(ssa_grad_norm(empty)) == 0.0 and float(ssa_clip_grad_norm(empty, 1.0)) == 0.0
