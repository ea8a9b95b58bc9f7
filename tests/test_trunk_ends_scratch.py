"""Scratch memory of a trunk's ends, asked of the built library on the CPU."""

import ctypes as C
import os

import pytest

from conftest import ROOT

trunk = pytest.importorskip("uor_fbs.trunk")
pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(ROOT, "uor-r4_amd", "lib", "libuor_trunk_hip.so")),
                                reason="the trunk library is not built")

SIZES = [(512, 1 << 20, 1024), (20000, 50000, 64), (262144, 32768, 256), (8192, 131072, 1024), (300, 1000, 100)]


def wanted(call, dtype, rows, vocab, width, **other):
    a = trunk.CHead(dtype=dtype, rows=rows, vocab=vocab, width=width, x_stride=width, w_stride=width, x=256, weight=256, **other)
    return getattr(trunk.lib(), f"uor_trunk_{call}_workspace_bytes")(C.byref(a))


@pytest.mark.parametrize("dtype", [0, 1], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,width", SIZES)
def test_one_gradient_wants_none_of_the_others(dtype, rows, vocab, width):
    """Beside what both need (G, rows and words laid out, a few numbers a row) dx needs nothing that goes by words x width, and
    dweight nothing that goes by rows x width but its sort's parts."""
    both = wanted("loss_backward", dtype, rows, vocab, width, dx=256, dweight=256)
    dx, dw = wanted("loss_backward", dtype, rows, vocab, width, dx=256), wanted("loss_backward", dtype, rows, vocab, width, dweight=256)
    assert 0 < dx <= both and 0 < dw <= both
    size = 4 if dtype else 2
    up = lambda v, to: (v + to - 1) // to * to  # noqa: E731
    all_rows, all_words = up(rows, 256), up(vocab, 256)
    laid = (2 * all_rows + vocab) * up(width * size, 64)
    slots, most_g = 160 << 20, min(1 << 30, all_rows * all_words * size)
    assert dx <= most_g + laid + slots + 4 * all_rows * up(width, 128) + 64 * all_rows
    assert dw <= most_g + laid + slots + 2 * 4 * all_words * up(width, 128) + all_words + 64 * all_rows + rows * width


@pytest.mark.parametrize("dtype", [0, 1], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,width", [*SIZES, (1 << 24, 9, 8), (1 << 20, 1000, 16), (1, 1, 1), (70, 1 << 23, 8192)])
def test_what_a_loss_and_an_embedding_want(dtype, rows, vocab, width):
    """x and weight by rows of whole 64 bytes, 40 bytes a row and 9 MB; 16 bytes a row, a quarter of dy in 32 bits and 1 MB."""
    row = (width * (4 if dtype else 2) + 63) // 64 * 64
    assert 0 < wanted("loss", dtype, rows, vocab, width, targets=256) <= ((rows + 255) // 256 * 256 + vocab) * row + 40 * (rows + 256) + (9 << 20)
    a = trunk.CEmbed(dtype=dtype, table_dtype=dtype, rows=rows, vocab=vocab, width=width, dy_stride=width, tokens=256, dy=256)
    assert 0 < trunk.lib().uor_trunk_embed_backward_workspace_bytes(C.byref(a)) <= 16 * rows + rows * width + 8 * width + (1 << 20) + (1 << 13)
