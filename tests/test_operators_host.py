"""The decoder-step operators' host side without a GPU: argument checks of the C entry points before
any CUDA call, workspace sizes, the ctypes mirrors of the header's structs, and the Python layer's
refusals of CPU tensors."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

REPO = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def lib():
    from SSA import _lib
    if not _lib.LIB_PATH.exists():
        import __graft_entry__
        __graft_entry__.build()
    return _lib.load()


def _ce(**kw):
    from SSA import _lib
    base = dict(dtype=2, rows=100, hidden=64, vocab=1000, x=256, x_stride=64, w=256, w_stride=64,
                targets=256, ignore_index=-100, reduction=1)
    base.update(kw)
    return _lib.SsaLinearCe(**base)


def _ffn(**kw):
    from SSA import _lib
    base = dict(dtype=2, rows=100, hidden=64, ffn=96, x=256, x_stride=64, w=256, w_stride=64)
    base.update(kw)
    return _lib.SsaGatedFfn(**base)


def _rope(**kw):
    from SSA import _lib
    base = dict(dtype=2, B=1, S=10, Hq=4, Hkv=2, D=64, qkv=_lib.SsaTensor(256, 0, 64, 512), cos=256,
                sin=256, table_rows=10, positions=None, positions_64=0, positions_stride=0,
                q_weight=None, k_weight=None, weight_dtype=2, eps=1e-5)
    base.update(kw)
    return _lib.SsaQkRope(**base)


def test_linear_ce_arguments(lib):
    from SSA import _lib
    for kw, code in ((dict(dtype=0), _lib.SSA_ERR_UNSUPPORTED), (dict(rows=0), _lib.SSA_ERR_BAD_SHAPE),
                     (dict(hidden=60), _lib.SSA_ERR_BAD_SHAPE),
                     (dict(rows=1 << 25), _lib.SSA_ERR_BAD_SHAPE),
                     (dict(reduction=3), _lib.SSA_ERR_UNSUPPORTED), (dict(x=None), _lib.SSA_ERR_NULL),
                     (dict(x=258), _lib.SSA_ERR_BAD_STRIDE), (dict(w_stride=68), _lib.SSA_ERR_BAD_STRIDE),
                     (dict(x_stride=56), _lib.SSA_ERR_BAD_STRIDE)):
        p = ctypes.byref(_ce(**kw))
        assert lib.ssa_linear_ce_fwd(p, 256, 256, 256, 256, 1 << 40, None) == code, kw
        assert lib.ssa_linear_ce_bwd(p, 256, 256, 256, 256, 256, 256, 1 << 40, None) == code, kw
        assert lib.ssa_linear_ce_fwd_workspace_size(p) == 0
    p = ctypes.byref(_ce())
    assert lib.ssa_linear_ce_fwd(p, None, 256, 256, 256, 1 << 40, None) == _lib.SSA_ERR_NULL
    assert lib.ssa_linear_ce_bwd(p, 256, 256, None, 256, 256, 256, 1 << 40, None) == _lib.SSA_ERR_NULL
    assert lib.ssa_linear_ce_bwd(p, 256, 256, 256, 264, 256, 256, 1 << 40, None) == _lib.SSA_ERR_BAD_STRIDE
    assert lib.ssa_linear_ce_bwd(p, 256, 256, 256, None, None, None, 0, None) == _lib.SSA_OK
    # no [rows, vocab] matrix: far below 16-bit logits once the vocabulary is walked in pieces
    big = _ce(rows=65536, vocab=131072, hidden=2048, x_stride=2048, w_stride=2048)
    assert lib.ssa_linear_ce_bwd_workspace_size(ctypes.byref(big)) < 2 * 65536 * 131072 // 10


def test_sizes_beyond_2_to_the_24(lib):
    from SSA import _lib
    big = (1 << 24) + 8
    for kw in (dict(rows=big), dict(hidden=big, x_stride=big, w_stride=big), dict(vocab=big)):
        p = ctypes.byref(_ce(**kw))
        assert lib.ssa_linear_ce_fwd(p, 256, 256, 256, 256, 1 << 40, None) == _lib.SSA_ERR_BAD_SHAPE
        assert lib.ssa_linear_ce_bwd_workspace_size(p) == 0
    for kw in (dict(rows=big), dict(hidden=big, x_stride=big, w_stride=big), dict(ffn=big)):
        p = ctypes.byref(_ffn(**kw))
        assert lib.ssa_gated_ffn_fwd(p, 256, 1 << 30, None) == _lib.SSA_ERR_BAD_SHAPE
        assert lib.ssa_gated_ffn_bwd_workspace_size(p) == 0


def test_gated_ffn_arguments(lib):
    from SSA import _lib
    for kw, code in ((dict(dtype=0), _lib.SSA_ERR_UNSUPPORTED), (dict(ffn=0), _lib.SSA_ERR_BAD_SHAPE),
                     (dict(hidden=4), _lib.SSA_ERR_BAD_SHAPE), (dict(w=None), _lib.SSA_ERR_NULL),
                     (dict(w=264), _lib.SSA_ERR_BAD_STRIDE), (dict(x_stride=60), _lib.SSA_ERR_BAD_STRIDE)):
        p = ctypes.byref(_ffn(**kw))
        assert lib.ssa_gated_ffn_fwd(p, 256, 96, None) == code, kw
        assert lib.ssa_gated_ffn_bwd(p, 256, 96, 256, 256, 256, 1 << 40, None) == code, kw
        assert lib.ssa_gated_ffn_bwd_workspace_size(p) == 0
    p = ctypes.byref(_ffn())
    assert lib.ssa_gated_ffn_fwd(p, 256, 95, None) == _lib.SSA_ERR_BAD_STRIDE
    assert lib.ssa_gated_ffn_bwd(p, None, 96, 256, 256, 256, 1 << 40, None) == _lib.SSA_ERR_NULL
    assert lib.ssa_gated_ffn_bwd_workspace_size(p) >= 2 * 100 * 2 * 96


def test_qk_rope_arguments(lib):
    from SSA import _lib
    T = _lib.SsaTensor
    good = T(256, 0, 64, 256)
    for kw, code in ((dict(D=48), _lib.SSA_ERR_UNSUPPORTED), (dict(S=0), _lib.SSA_ERR_BAD_SHAPE),
                     (dict(table_rows=0), _lib.SSA_ERR_BAD_SHAPE), (dict(cos=None), _lib.SSA_ERR_NULL),
                     (dict(cos=260), _lib.SSA_ERR_BAD_STRIDE), (dict(q_weight=256), _lib.SSA_ERR_NULL),
                     (dict(qkv=T(256, 0, 60, 512)), _lib.SSA_ERR_BAD_STRIDE),
                     (dict(qkv=T(None, 0, 64, 512)), _lib.SSA_ERR_NULL),
                     (dict(weight_dtype=1), _lib.SSA_ERR_UNSUPPORTED)):
        p = ctypes.byref(_rope(**kw))
        assert lib.ssa_qk_rope_fwd(p, 256, 256, None) == code, kw
        assert lib.ssa_qk_rope_bwd(p, good, good, good, 256, None, None, None, 0, None) == code, kw
    p = ctypes.byref(_rope(q_weight=256, k_weight=256))
    assert lib.ssa_qk_rope_bwd_workspace_size(p) > 0
    assert lib.ssa_qk_rope_bwd(p, good, good, good, 256, 256, 256, None, 0, None) == _lib.SSA_ERR_WORKSPACE


def test_grad_list_arguments(lib):
    from SSA import _lib
    from array import array

    def lst(ptrs, sizes, outs=None, dtype=0, out_dtype=0):
        arr = [array("q", ptrs), array("q", sizes), array("q", outs) if outs else None]
        p = _lib.SsaGradList(dtype, len(sizes), arr[0].buffer_info()[0], arr[1].buffer_info()[0],
                             arr[2].buffer_info()[0] if outs else None, out_dtype)
        p.keep = arr
        return p

    def clip(p, norm=256, max_norm=1.0):
        return lib.ssa_grad_clip(ctypes.byref(p), max_norm, norm, 256, 1 << 40, None)

    bad, null = _lib.SSA_ERR_BAD_SHAPE, _lib.SSA_ERR_NULL
    assert clip(lst([4096, 4096], [4, 4])) == bad                      # the same tensor twice
    assert clip(lst([4096, 4104], [4, 4])) == bad                      # a view of it
    assert clip(lst([4096], [4], [4100])) == bad                       # an output inside its gradient
    assert clip(lst([4096, 8192], [4, 4], [16384, 16384])) == bad
    assert clip(lst([4096], [4], [4096], dtype=2, out_dtype=0)) == bad  # wider than what it replaces
    assert clip(lst([4096], [4], [8192], dtype=2, out_dtype=1)) == _lib.SSA_ERR_UNSUPPORTED
    assert clip(lst([4098], [4])) == _lib.SSA_ERR_BAD_STRIDE
    assert clip(lst([0], [4])) == null
    assert clip(lst([4096], [-1])) == bad and clip(lst([4096], [4]), max_norm=-1.0) == bad
    assert clip(lst([4096], [4]), norm=None) == null
    assert lib.ssa_grad_clip_workspace_size(ctypes.byref(lst([4096, 0], [100000, 0]))) >= 8 * 7


def test_ctypes_structs_match_the_c_header(tmp_path):
    from SSA import _lib
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    structs = {"ssa_linear_ce_t": _lib.SsaLinearCe, "ssa_gated_ffn_t": _lib.SsaGatedFfn,
               "ssa_qk_rope_t": _lib.SsaQkRope, "ssa_grad_list_t": _lib.SsaGradList}
    prog = ["#include <stdio.h>", "#include <stddef.h>", '#include "ssa_b200.h"', "int main(void) {"]
    for c, py in structs.items():
        prog.append(f'  printf("{c} %zu\\n", sizeof({c}));')
        prog += [f'  printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(prog + ["  return 0;", "}"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True,
                                                       check=True).stdout.splitlines())
    for c, py in structs.items():
        assert int(out[c]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert int(out[f"{c}.{f}"]) == getattr(py, f).offset, (c, f)


def test_python_layer_rejects_cpu_tensors():
    from SSA.ssa_cross_entropy import ssa_linear_cross_entropy
    from SSA.ssa_gated_ffn import ssa_gated_ffn
    from SSA.ssa_grad_clip import ssa_clip_grad_norm, ssa_grad_norm
    from SSA.ssa_qk_norm_rope import ssa_qk_norm_rope
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.long)
    table = torch.zeros(4, 16)
    for call in (lambda: ssa_linear_cross_entropy(x, x, t), lambda: ssa_gated_ffn(x, x),
                 lambda: ssa_qk_norm_rope(x, 2, 1, table, table), lambda: ssa_grad_norm([x]),
                 lambda: ssa_clip_grad_norm([x], 1.0)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
