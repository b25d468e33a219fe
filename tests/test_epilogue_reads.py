"""Reads of accumulators in the tensor-core products' epilogues: each one that is started is waited for
before the tile goes back to the MMAs, which overwrite what is still being read. On the CPU the
sources are read for a way out between a read and its wait; on the GPU the feed-forward runs with
inner sizes whose last tile leaves a warp without columns, over several tiles a cluster."""

import re
from pathlib import Path

import pytest
import torch

CSRC = Path(__file__).resolve().parent.parent / "luciole-1b_b200" / "csrc"


def _block(text, start):
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[start:i + 1]
    raise AssertionError("unbalanced braces")


def test_no_way_out_between_a_read_and_its_wait():
    seen = 0
    for f in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", f.read_text())
        for m in re.finditer(r"struct (Epi\w+) \{", text):
            struct = _block(text, m.end() - 1)
            tile = re.search(r"void tile\(", struct)
            body = _block(struct, struct.index("{", tile.start()))
            after = body[body.index("e.fetch("):]
            seen += 1
            assert not re.search(r"\b(break|return|goto)\b", after), (f.name, m.group(1))
            assert after.rindex("e.settle(") > 0
    assert seen >= 5


@pytest.mark.gpu
@pytest.mark.parametrize("f", [1281, 1312, 1313, 1344, 1345, 1377])
def test_last_tile_without_columns_for_a_warp(cuda_device, f):
    """More tiles than clusters, and the last of a row with 1 to 97 of its 128 columns."""
    from test_gpu_gated_ffn import _check, _data
    _check(*_data(3000, 264, f, torch.bfloat16, f, cuda_device))
