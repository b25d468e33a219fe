"""Paths of the decoder-step operators that only large calls take, or several at once: the rotation's
eight heads a lane with streaming stores, the loss over several pieces of the vocabulary whose dx is
split as well, two streams, and sums of squares held to their own roundings."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm,dtype", [(False, torch.bfloat16), (True, torch.bfloat16),
                                        (True, torch.float32)])
@pytest.mark.parametrize("lead,hq,hkv", [((76001,), 13, 3), ((3, 22003), 17, 1)])
def test_rotation_of_many_tokens(cuda_device, norm, dtype, lead, hq, hkv):
    """78 and 76 million query and key elements: eight heads a lane forward, four backward, head counts
    that neither divides, results that do not stay in L2."""
    from test_gpu_qk_norm_rope import _check
    _check(lead, hq, hkv, 64, dtype, cuda_device, norm, seed=hq)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_pieces_of_the_vocabulary_with_split_contractions(cuda_device, reduction):
    """Four pieces, the last narrower, and dx summed over two splits of each."""
    from test_gpu_linear_ce import _check, _data
    _check(*_data(4100, 1024, 128001, torch.bfloat16, 33, 0.1, cuda_device), reduction)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_more_rows_than_a_piece_of_256_mib_takes(cuda_device, reduction):
    """140,001 rows: pieces of the least width, 1024 columns, are larger than that."""
    from test_gpu_linear_ce import _check, _data
    _check(*_data(140001, 64, 2101, torch.bfloat16, 35, 0.1, cuda_device), reduction)


def _ffn(seed, dev):
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    from test_gpu_gated_ffn import _data
    x, w, dh = _data(700, 264, 1365, torch.bfloat16, seed, dev)

    def run():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        h = ssa_gated_ffn(a, b)
        return [h.detach(), *torch.autograd.grad(h, (a, b), dh)]
    return run


def _rope(seed, dev):
    import luciole_train as LT
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    g = torch.Generator(device=dev).manual_seed(seed)
    qkv = torch.randn(5000, 20 * 64, generator=g, device=dev).bfloat16()
    ws = [torch.rand(64, generator=g, device=dev).bfloat16() for _ in range(2)]
    cos, sin = LT.rope_tables(5000, 64, 1e4, dev)
    grads = [torch.randn(5000, n, 64, generator=g, device=dev).bfloat16() for n in (12, 4, 4)]

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (qkv, *ws)]
        out = ssa_qk_norm_rope(leaves[0], 12, 4, cos, sin, *leaves[1:])
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, grads)]
    return run


def _clip(seed, dev):
    from SSA.ssa_grad_clip import ssa_clip_grad_norm
    g = torch.Generator(device=dev).manual_seed(seed)
    grads = [torch.randn(s, generator=g, device=dev).bfloat16() for s in (3_000_001, 7, 500_000)]

    def run():
        out = [torch.empty_like(t, dtype=torch.float32) for t in grads]
        mine = [t.clone() for t in grads]
        return [ssa_clip_grad_norm(grads, 1.0, out=out), *out, ssa_clip_grad_norm(mine, 2.0), *mine]
    return run


@pytest.mark.parametrize("make", [_ffn, _rope, _clip])
def test_two_streams_at_once(cuda_device, make):
    runs = [make(seed, cuda_device) for seed in (1, 2)]
    want = [run() for run in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, (st, run) in enumerate(zip(streams, runs)):
            with torch.cuda.stream(st):
                got[i] = run()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


# The squares of a 16-byte load are added in pairs in fp32: at most three roundings on each (fp32: y y,
# the pair's multiply-add, one sum; 16-bit types: their squares are exact, the multiply-add, two sums),
# everything above in fp64. The root halves that, and the norm is rounded once.
NORM_STEPS = 3 / 2 + 1


@pytest.mark.parametrize("pattern,dtype", [
    # patterns whose rounding errors all have one sign when the squares are added one after another
    # in fp32 over a thread's 32 or 64 elements: 2.6 and 3.8 steps off then
    ([0.06341463327407837, 0.0017083704005926847, 0.00876022782176733, 0.0015683879610151052],
     torch.float32),
    ([0.0634765625, 0.0012664794921875, 0.0034637451171875, 0.0030670166015625,
      0.0027008056640625, 0.0014190673828125, 0.0025177001953125, 0.003997802734375],
     torch.bfloat16)])
@pytest.mark.parametrize("repeats", [1, 2048, 123457])
def test_norm_of_a_repeated_pattern(cuda_device, pattern, dtype, repeats):
    from SSA.ssa_grad_clip import ssa_grad_norm
    g = torch.tensor(pattern).to(dtype).to(cuda_device).repeat(repeats)
    want = math.sqrt(float(g.double().square().sum()))
    assert abs(float(ssa_grad_norm([g])) - want) <= (NORM_STEPS * 2.0 ** -24 + 1e-12) * want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_and_factor_to_their_own_roundings(cuda_device, dtype):
    """The factor is formed in fp64 from the sum and rounded once; an element times it in fp32, once."""
    from SSA.ssa_grad_clip import ssa_clip_grad_norm, ssa_grad_norm
    for seed in range(20):
        gen = torch.Generator(device=cuda_device).manual_seed(seed)
        grads = [(torch.randn(n, generator=gen, device=cuda_device) * 0.01).to(dtype)
                 for n in (100_003, 16, 40_000)]
        want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        lim = (NORM_STEPS * 2.0 ** -24 + 1e-12) * want
        assert abs(float(ssa_grad_norm(grads)) - want) <= lim
        out = [torch.empty_like(g, dtype=torch.float32) for g in grads]
        norm = ssa_clip_grad_norm(grads, 0.37 * want, out=out)
        assert abs(float(norm) - want) <= lim
        coef = 0.37 * want / (want + 1e-6)
        for g, o in zip(grads, out):
            exact = g.double() * coef
            assert ((o.double() - exact).abs() <=
                    ((NORM_STEPS + 1) * 2.0 ** -24 + 1e-12) * exact.abs()).all()
