"""Sizes that do not fit the C structs' fields are refused: wrapped, a call would take another size's
work for its own and leave the rest of its results unwritten. Tensors without data (meta)."""

import pytest
import torch

BIG = (1 << 32) + 8


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, device="meta", dtype=dtype)


def test_matrix_operators():
    from SSA import ssa_cross_entropy as ce, ssa_gated_ffn as ffn
    t = _meta(8, dtype=torch.int64)
    ce._problem(_meta(8, 8), _meta(16, 8), t, -100, 1)
    ffn._problem(_meta(8, 8), _meta(16, 8))
    for x, w in ((_meta(BIG, 8), _meta(16, 8)), (_meta(8, BIG), _meta(16, BIG)),
                 (_meta(8, 8), _meta(2 * BIG, 8))):
        with pytest.raises(ValueError, match="32 bits"):
            ce._problem(x, w, t, -100, 1)
        with pytest.raises(ValueError, match="32 bits"):
            ffn._problem(x, w)


def test_rotation():
    from SSA import ssa_qk_norm_rope as rope
    f32 = torch.float32

    def problem(b, s, rows=64):
        return rope._problem(_meta(b, s, 4, 16), 2, 1, _meta(rows, 16, dtype=f32),
                             _meta(rows, 16, dtype=f32), None, 0, None, None, 1e-5)

    problem(2, 8)
    for args in ((BIG, 1), (1, BIG), (1, 8, BIG)):
        with pytest.raises(ValueError, match="32 bits"):
            problem(*args)


@pytest.mark.gpu
def test_ignore_index(cuda_device):
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    x, w = (torch.zeros(n, 8, device=cuda_device, dtype=torch.bfloat16) for n in (4, 16))
    t = torch.zeros(4, device=cuda_device, dtype=torch.int64)
    ssa_linear_cross_entropy(x, w, t, ignore_index=-(1 << 63))
    for bad in (1 << 63, (1 << 64) - 100):
        with pytest.raises(ValueError, match="64 bits"):
            ssa_linear_cross_entropy(x, w, t, ignore_index=bad)
