"""A trunk's ends over its vocabulary, on the CPU: the oracle's gradients against differences, and the refusals of
uor_fbs.trunk and of the C ABI."""

import ctypes as C
import os

import pytest
import torch

import ends_cases as oracle
from conftest import ROOT

trunk = pytest.importorskip("uor_fbs.trunk")
built = pytest.mark.skipif(not os.path.exists(os.path.join(ROOT, "uor-r4_amd", "lib", "libuor_trunk_hip.so")),
                           reason="the trunk library is not built")


def differences(function, x, got, step=1e-6):
    flat = x.reshape(-1)
    for i in range(flat.numel()):
        at = []
        for sign in (1, -1):
            moved = flat.clone()
            moved[i] += sign * step
            at.append(function(moved.reshape(x.shape)))
        assert abs((at[0] - at[1]) / (2 * step) - got.reshape(-1)[i]) < 1e-6 * (1 + abs(got.reshape(-1)[i])), i


def test_the_loss_gradients_are_the_differences():
    g = torch.Generator().manual_seed(3)
    normal = lambda *shape: torch.randn(shape, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, targets = normal(5, 4), normal(7, 4), torch.tensor([3, -1, 0, 6, 7])
    da, db = normal(5), normal(5)
    dx, dw = oracle.loss_backward(da, x, w, targets, db)

    def total(x, w):
        losses, lse = oracle.loss(x, w, targets)
        return ((losses * da).sum() + (lse * db).sum()).item()

    differences(lambda v: total(v, w), x, dx)
    differences(lambda v: total(x, v), w, dw)


def test_the_embedding_gradient_is_the_differences():
    g = torch.Generator().manual_seed(4)
    table, dy = torch.randn(6, 3, generator=g, dtype=torch.float64), torch.randn(5, 3, generator=g, dtype=torch.float64)
    tokens = torch.tensor([2, 5, -1, 2, 6])
    differences(lambda v: (oracle.embed(tokens, v, 1.5) * dy).sum().item(), table, oracle.embed_backward(dy, tokens, 6, 1.5)[0])


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int64)


EMBED_REFUSALS = [
    ((ints(4), bf16(10, 8)), {}, "on cpu"),
    (([0, 1], bf16(10, 8)), {}, "tokens is no tensor"),
    ((torch.zeros(4), bf16(10, 8)), {}, "tokens is torch.float32"),
    ((ints(2, 2), bf16(10, 8)), {}, "tokens has shape"),
    ((ints(4), bf16(10)), {}, "axes word and value"),
    ((ints(4), bf16(0, 8)), {}, "table of 0 words"),
    ((ints(4), bf16(10, 8193)), {}, "at most"),
    ((ints(4), torch.zeros(10, 8, dtype=torch.float16)), {}, "table is no tensor of bfloat16 or float32"),
    ((ints(4), None), {}, "table is no tensor"),
]


@pytest.mark.parametrize("args,kw,text", EMBED_REFUSALS, ids=[t for *_, t in EMBED_REFUSALS])
def test_embed_refuses(args, kw, text):
    with pytest.raises(trunk.TrunkError, match=text):
        trunk.embed(*args, **kw)
    with pytest.raises(trunk.TrunkError, match=text):
        trunk.embed_backward(bf16(4, 8), *args, **kw)


def test_embed_refuses_types_and_rows():
    with pytest.raises(trunk.TrunkError, match="dtype is torch.float16"):
        trunk.embed(ints(4), bf16(10, 8), dtype=torch.float16)
    for dy, text in ((None, "dy is no tensor"), (bf16(3, 8), "dy has shape"), (bf16(4, 9), "dy has shape")):
        with pytest.raises(trunk.TrunkError, match=text):
            trunk.embed_backward(dy, ints(4), bf16(10, 8))


HEAD_REFUSALS = [
    ((bf16(4, 8), bf16(10, 8), ints(4)), "on cpu"),
    ((bf16(4, 8), bf16(10, 9), ints(4)), "x has shape"),
    ((torch.zeros(4, 8), bf16(10, 8), ints(4)), "x is torch.float32"),
    ((bf16(4, 2, 4), bf16(10, 8), ints(4)), "x has the axes"),
    ((bf16(4, 8), bf16(10, 8, 1), ints(4)), "axes word and value"),
    ((bf16(4, 8), bf16(0, 8), ints(4)), "weight of 0 words"),
    ((bf16(4, 8), bf16(10, 8), ints(5)), "targets has shape"),
    ((bf16(4, 8), bf16(10, 8), torch.zeros(4)), "targets is torch.float32"),
    ((bf16(4, 8), bf16(10, 8), None), "targets is no tensor"),
    ((bf16(4, 8), bf16(10, 8), [1, 2, 3, 4]), "targets is no tensor"),
]


@pytest.mark.parametrize("args,text", HEAD_REFUSALS, ids=[f"{i}-{t}" for i, (_, t) in enumerate(HEAD_REFUSALS)])
def test_loss_refuses(args, text):
    with pytest.raises(trunk.TrunkError, match=text):
        trunk.loss(*args)
    with pytest.raises(trunk.TrunkError, match=text):
        trunk.loss_backward(torch.zeros(4), *args, torch.zeros(4))
    if "targets" not in text:
        with pytest.raises(trunk.TrunkError, match=text):
            trunk.choose(*args[:2])


def test_loss_backward_refuses():
    args = bf16(4, 8), bf16(10, 8), ints(4)
    for da, lse, kw, text in ((torch.zeros(5), torch.zeros(4), {}, "dlosses has shape"), (torch.zeros(4), None, {}, "lse is no tensor"),
                              (torch.zeros(4), torch.zeros(4).double(), {}, "lse is torch.float64"),
                              (None, torch.zeros(4), dict(dlse=bf16(4)), "dlse is torch.bfloat16"),
                              (None, torch.zeros(4), dict(dtype=torch.float16), "dtype is torch.float16")):
        with pytest.raises(trunk.TrunkError, match=text):
            trunk.loss_backward(da, *args, lse, **kw)


@built
def test_c_entries_refuse_before_they_reach_a_device():
    L = trunk.lib()
    last = lambda: L.uor_trunk_last_error().decode()  # noqa: E731
    some = 1 << 20  # never read: the refusals come first

    def head(**change):
        return trunk.CHead(**{**dict(rows=5, vocab=9, width=8, x_stride=8, w_stride=8, x=some, weight=some, targets=some, losses=some, lse=some,
                                     tokens=some, logprobs=some, dx=some, dweight=some), **change})

    calls = (L.uor_trunk_loss_async, L.uor_trunk_loss_backward_async, L.uor_trunk_choose_async)
    for change, text in [(dict(dtype=2), "dtype"), (dict(width=0), "width"), (dict(width=8193), "width"), (dict(vocab=0), "vocabulary"),
                         (dict(vocab=(1 << 23) + 1), "vocabulary"), (dict(rows=(1 << 24) + 1), "rows"), (dict(x_stride=7), "overlap"),
                         (dict(w_stride=7), "overlap"), (dict(x=None), "null x"), (dict(weight=None), "null x or weight")]:
        for call in calls:
            assert call(C.byref(head(**change)), None, 0, None) == -1 and text in last(), (change, last())
    for change, call, text in [(dict(targets=None), 0, "targets"), (dict(lse=None), 0, "lse"), (dict(targets=None), 1, "targets"),
                               (dict(lse=None), 1, "lse"), (dict(dweight_dtype=2), 1, "dweight_dtype"), (dict(tokens=None), 2, "tokens")]:
        assert calls[call](C.byref(head(**change)), None, 0, None) == -1 and text in last(), (change, last())
    for call, size in zip(calls, (L.uor_trunk_loss_workspace_bytes, L.uor_trunk_loss_backward_workspace_bytes, L.uor_trunk_choose_workspace_bytes)):
        a = head()
        want = size(C.byref(a))
        assert want > 0
        for workspace, n in ((None, want), (some, want - 1), (some + 16, want)):
            assert call(C.byref(a), workspace, n, None) == -1 and "workspace" in last()
        assert call(None, None, 0, None) == -1 and "null" in last()

    def embed(**change):
        return trunk.CEmbed(**{**dict(rows=5, vocab=9, width=8, scale=1.0, table_stride=8, dy_stride=8, tokens=some, table=some, y=some, dy=some,
                                      dtable=some), **change})

    for change, text in [(dict(dtype=2), "dtype"), (dict(table_dtype=2), "dtype"), (dict(width=0), "width"), (dict(vocab=0), "vocabulary"),
                         (dict(rows=(1 << 24) + 1), "rows"), (dict(tokens=None), "tokens")]:
        a = embed(**change)
        assert L.uor_trunk_embed_async(C.byref(a), None) == -1 and text in last(), (change, last())
        assert L.uor_trunk_embed_backward_async(C.byref(a), None, 0, None) == -1 and text in last(), (change, last())
    assert L.uor_trunk_embed_async(C.byref(embed(table_stride=7)), None) == -1 and "overlap" in last()
    assert L.uor_trunk_embed_async(C.byref(embed(y=None)), None) == -1 and "null" in last()
    assert L.uor_trunk_embed_backward_async(C.byref(embed(dy_stride=7)), None, 0, None) == -1 and "overlap" in last()
    assert L.uor_trunk_embed_backward_async(C.byref(embed(dtable=None)), None, 0, None) == -1 and "null" in last()
    assert L.uor_trunk_embed_backward_async(C.byref(embed()), None, 0, None) == -1 and "workspace" in last()


@built
@pytest.mark.parametrize("rows,vocab,width", [(32768, 32768, 256), (262144, 32768, 256), (8192, 131072, 1024), (1 << 20, 131072, 512), (1 << 20, 1 << 23, 64)])
def test_scratch_memory_does_not_grow_with_the_logits(rows, vocab, width):
    """A piece of the logits' gradient is of 2^30 bytes at most; the rest goes by rows x width and by words x width."""
    L = trunk.lib()
    a = trunk.CHead(dtype=0, rows=rows, vocab=vocab, width=width, x_stride=width, w_stride=width, x=16, weight=16)
    # Sums so far of 32 bits: dx's and dW's in up to 512 tiles' worth of splits, or of one piece of the one and all of the other,
    # and the targets' terms; the matrix and the rows laid out; the sort and its parts.
    laid = 2 * width * (vocab + 2 * rows)
    most = (1 << 30) + 4 * 2 * max(rows * width, 512 * 256 * 128) + 4 * 3 * max(vocab * width, 512 * 256 * 128) + laid
    most += rows * width // 8 + rows * 64 + (1 << 22)
    assert 0 < L.uor_trunk_loss_backward_workspace_bytes(C.byref(a)) <= most
    # Two sums of a row for each part of the words: 2,048 blocks' worth, or one part.
    assert 0 < L.uor_trunk_loss_workspace_bytes(C.byref(a)) <= laid + rows * 16 + 32 * (max(rows, 2048 * 128) + (1 << 16))


def test_the_struct_sizes_are_the_librarys():
    assert (C.sizeof(trunk.CEmbed), C.sizeof(trunk.CHead)) == (32 + 2 * 8 + 5 * 8, 32 + 2 * 8 + 11 * 8)
