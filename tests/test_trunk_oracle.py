"""The oracle of the float trunk's operators: its gradients against central differences, and the
refusals of uor_fbs.trunk and of the C ABI, all on the CPU."""

import ctypes as C
import os

import pytest
import torch

import trunk_cases as oracle
from conftest import ROOT

trunk = pytest.importorskip("uor_fbs.trunk")
LIB = os.path.join(ROOT, "uor-r4_amd", "lib", "libuor_trunk_hip.so")
built = pytest.mark.skipif(not os.path.exists(LIB), reason="the trunk library is not built")


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, dtype=torch.float64)


def differences(function, inputs, name, got, step=1e-6):
    """got against central differences of function(**inputs) at the named input."""
    x = inputs[name]
    flat = x.reshape(-1)
    for i in range(flat.numel()):
        at = []
        for sign in (1, -1):
            moved = flat.clone()
            moved[i] += sign * step
            at.append(function(**{**inputs, name: moved.reshape(x.shape)}))
        assert abs((at[0] - at[1]) / (2 * step) - got.reshape(-1)[i]) < 1e-6 * (1 + abs(got.reshape(-1)[i])), (name, i)


def test_scan_gradients_are_the_differences():
    g = torch.Generator().manual_seed(3)
    off = oracle.offsets_of([4, 0, 3])
    x = dict(x=normal(g, 7, 4, 3), dt=normal(g, 7, 4), A=-normal(g, 4).abs(), B=normal(g, 7, 2, 2), C=normal(g, 7, 2, 2),
             D=normal(g, 4), dt_bias=normal(g, 4), initial=normal(g, 3, 4, 3, 2))
    dy, dfinal = normal(g, 7, 4, 3), normal(g, 3, 4, 3, 2)
    got = oracle.scan_backward(dy, x["x"], x["dt"], x["A"], x["B"], x["C"], x["D"], x["dt_bias"], off, x["initial"], dfinal)

    def loss(**v):
        y, final = oracle.scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["dt_bias"], off, v["initial"])
        return ((y * dy).sum() + (final * dfinal).sum()).item()

    for name in x:
        differences(loss, x, name, got["d" + name])


@pytest.mark.parametrize("silu", [True, False])
def test_conv_gradients_are_the_differences(silu):
    g = torch.Generator().manual_seed(4)
    off = oracle.offsets_of([2, 0, 5, 1])
    x = dict(x=normal(g, 8, 3), weight=normal(g, 3, 4), bias=normal(g, 3), initial=normal(g, 4, 3, 3))
    dy, dfinal = normal(g, 8, 3), normal(g, 4, 3, 3)
    got, _ = oracle.conv_backward(dy, x["x"], x["weight"], x["bias"], off, x["initial"], dfinal, silu)

    def loss(**v):
        y, final, _ = oracle.conv(v["x"], v["weight"], v["bias"], off, v["initial"], silu)
        return ((y * dy).sum() + (final * dfinal).sum()).item()

    for name in x:
        differences(loss, x, name, got["d" + name])


@pytest.mark.parametrize("absent", [(), ("gate",), ("post", "scale"), ("residual",), ("out", "gate", "post", "scale")])
def test_norm_gradients_are_the_differences(absent):
    g = torch.Generator().manual_seed(5)
    x = dict(residual=normal(g, 3, 5), out=normal(g, 3, 5), gate=normal(g, 3, 5), post=normal(g, 5), scale=normal(g, 5), pre=normal(g, 5))
    x = {k: None if k in absent else v for k, v in x.items()}
    dr, dn = normal(g, 3, 5), normal(g, 3, 5)
    got, _ = oracle.norms_backward(dr, dn, **x)

    def loss(**v):
        r, n = oracle.norms(**v)
        return ((r * dr).sum() + (n * dn).sum()).item()

    for name in x:
        if x[name] is not None:
            differences(loss, x, name, got["d" + name])


# ---------------------------------------------------------------------------------------------
# Refusals.


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def f32(*shape):
    return torch.zeros(shape)


def scan_inputs(**other):
    x = dict(x=bf16(5, 4, 8), dt=bf16(5, 4), A=f32(4), B=bf16(5, 2, 6), C=bf16(5, 2, 6))
    return {**x, **other}


SCAN_REFUSALS = [
    (dict(), "on cpu"),
    (dict(x=torch.zeros(5, 4, 8, dtype=torch.float16)), "x is no tensor of bfloat16 or float32"),
    (dict(x=bf16(5, 32)), "x has the axes"),
    (dict(dt=f32(5, 4)), "dt is torch.float32"),
    (dict(dt=bf16(4, 4)), "dt has shape"),
    (dict(A=bf16(4)), "A is torch.bfloat16"),
    (dict(A=None), "A is no tensor"),
    (dict(B=bf16(5, 3, 6)), "whole groups"),
    (dict(C=bf16(5, 2, 5)), "C has shape"),
    (dict(x=bf16(5, 4, 129)), "outside 1..128"),
    (dict(B=bf16(5, 2, 129)), "outside 1..128"),
    (dict(D=f32(5)), "D has shape"),
    (dict(offsets=torch.zeros(1, dtype=torch.int32)), "offsets has one place more"),
    (dict(offsets=torch.zeros(3)), "offsets is torch.float32"),
    (dict(offsets=torch.zeros(3, dtype=torch.int32), initial=f32(3, 4, 8, 6)), "initial has shape"),
]


@pytest.mark.parametrize("change,text", SCAN_REFUSALS, ids=[t for _, t in SCAN_REFUSALS])
def test_scan_refuses(change, text):
    with pytest.raises(trunk.TrunkError, match=text):
        trunk.scan(**scan_inputs(**change))
    with pytest.raises(trunk.TrunkError, match=text):
        trunk.scan_backward(bf16(5, 4, 8), **scan_inputs(**change))


def test_gradients_and_steps_refuse():
    with pytest.raises(trunk.TrunkError, match="dy has shape"):
        trunk.scan_backward(bf16(5, 4, 7), **scan_inputs())
    with pytest.raises(trunk.TrunkError, match="dy is no tensor"):
        trunk.scan_backward(None, **scan_inputs())
    with pytest.raises(trunk.TrunkError, match="dfinal has shape"):
        trunk.scan_backward(bf16(5, 4, 8), **scan_inputs(), dfinal=f32(2, 4, 8, 6))
    for states in (f32(5, 4, 8, 5), torch.zeros(5, 4, 8, 6, dtype=torch.float64), f32(5, 4, 6, 8).transpose(2, 3), None):
        with pytest.raises(trunk.TrunkError, match="states is no dense"):
            trunk.scan_step(**scan_inputs(), states=states)
    with pytest.raises(trunk.TrunkError, match="5 rows for 4 states"):
        trunk.scan_step(**scan_inputs(), states=f32(4, 4, 8, 6))
    with pytest.raises(trunk.TrunkError, match="slots has shape"):
        trunk.scan_step(**scan_inputs(), states=f32(4, 4, 8, 6), slots=torch.zeros(4, dtype=torch.int32))


def test_conv_refuses():
    x, w = bf16(6, 10), f32(10, 4)
    for args, text in [((x, w), "on cpu"), ((x, f32(10, 5)), "outside 1..4"), ((x, f32(9, 4)), "weight has shape"),
                       ((x, w, f32(9)), "bias has shape"), ((bf16(6, 2, 5), w), "x has the axes")]:
        with pytest.raises(trunk.TrunkError, match=text):
            trunk.conv(*args)
        with pytest.raises(trunk.TrunkError, match=text):
            trunk.conv_backward(bf16(*args[0].shape), *args)
    with pytest.raises(trunk.TrunkError, match="initial has shape"):
        trunk.conv(x, w, initial=bf16(1, 4, 10))
    with pytest.raises(trunk.TrunkError, match="states is no dense"):
        trunk.conv_step(x, w, f32(6, 3, 10))


def test_norms_refuse():
    r = bf16(4, 16)
    for args, kw, text in [((r, r), {}, "on cpu"), ((r,), {}, "nothing to compute"), ((r,), dict(gate=r, pre=f32(16)), "without a block"),
                           ((r, bf16(4, 15)), {}, "out has shape"), ((r, r), dict(post=bf16(16)), "post is torch.bfloat16"),
                           ((r, r), dict(eps=-1.0), "eps is negative"), ((bf16(4, 8193),), dict(pre=f32(8193)), "outside 1..")]:
        with pytest.raises(trunk.TrunkError, match=text):
            trunk.norms(*args, **kw)
    with pytest.raises(trunk.TrunkError, match="dnormed without pre"):
        trunk.norms_backward(r, r, r, r)


@built
def test_c_entries_refuse_before_they_reach_a_device():
    L = trunk.lib()
    for name in trunk.SYMBOLS:
        assert getattr(L, name)
    last = lambda: L.uor_trunk_last_error().decode()  # noqa: E731
    some = 1 << 20  # never read: the refusals come first

    def scan_args(**change):
        v = dict(dtype=0, tokens=5, seqs=1, heads=4, groups=2, dim=8, state=6, x_stride=32, dt_stride=4, b_stride=12, c_stride=12,
                 y_stride=32, x=some, dt=some, B=some, C=some, A=some, y=some)
        return trunk.CScan(**{**v, **change})

    for change, text in [(dict(dtype=2), "dtype"), (dict(groups=3), "whole groups"), (dict(dim=0), "dim"), (dict(state=200), "state"),
                         (dict(seqs=0), "sequences"), (dict(seqs=2), "without offsets"), (dict(x=None), "null rows"),
                         (dict(A=None), "null A"), (dict(x_stride=31), "overlap"), (dict(tokens=0x7fffffff), "too many"),
                         (dict(y=None), "null y")]:
        a = scan_args(**change)
        assert L.uor_trunk_scan_async(C.byref(a), None, 0, None) == -1 and text in last(), (change, last())
    a = scan_args(tokens=100_000)
    want = L.uor_trunk_scan_workspace_bytes(C.byref(a))
    assert want > 0
    for workspace, size in ((None, want), (some, want - 1), (some + 8, want)):
        assert L.uor_trunk_scan_async(C.byref(a), workspace, size, None) == -1 and "workspace" in last()
    a = scan_args()
    assert L.uor_trunk_scan_backward_async(C.byref(a), None, 0, None) == -1 and "null dy" in last()
    assert L.uor_trunk_scan_step_async(C.byref(a), None) == -1 and "states" in last()
    a = scan_args(states=some, slots=4)
    assert L.uor_trunk_scan_step_async(C.byref(a), None) == -1 and "5 rows for 4" in last()
    assert L.uor_trunk_scan_async(None, None, 0, None) == -1 and "null" in last()
    c = trunk.CConv(tokens=4, seqs=1, channels=8, taps=5, x_stride=8, y_stride=8, x=some, weight=some, y=some)
    assert L.uor_trunk_conv_async(C.byref(c), None) == -1 and "taps" in last()
    n = trunk.CNorms(rows=4, width=8, residual_stride=8, residual=some)
    assert L.uor_trunk_norms_async(C.byref(n), None) == -1 and "nothing" in last()


def test_the_struct_sizes_are_the_librarys():
    assert (C.sizeof(trunk.CScan), C.sizeof(trunk.CConv), C.sizeof(trunk.CNorms)) == (40 + 5 * 8 + 23 * 8, 32 + 2 * 8 + 15 * 8, 24 + 3 * 8 + 16 * 8)


def test_places_of_64_bits_stay_where_they_are_or_outside():
    """Slots and offsets may be int64; those past 32 bits become none that there is."""
    wide = torch.tensor([0, 5, -1, 1 << 31, 1 << 32, (1 << 32) + 5, -(1 << 32), 1 << 62])
    got = trunk._int32("slots", wide)
    most = 2 ** 31 - 1
    assert got.dtype == torch.int32 and got.tolist() == [0, 5, -1, most, most, most, -1, most]


def test_places_that_are_no_tensors_are_refused():
    x, w = bf16(6, 10), f32(10, 4)
    for call in (lambda: trunk.scan(**scan_inputs(offsets=[0, 5])), lambda: trunk.conv(x, w, offsets=[0, 6]),
                 lambda: trunk.conv_backward(x, x, w, offsets=(0, 6))):
        with pytest.raises(trunk.TrunkError, match="offsets is no tensor"):
            call()
    for call in (lambda: trunk.scan_step(**scan_inputs(), states=f32(6, 4, 8, 6), slots=[0, 1, 2, 3, 4]),
                 lambda: trunk.conv_step(x, w, bf16(6, 3, 10), slots=list(range(6)))):
        with pytest.raises(trunk.TrunkError, match="slots is no tensor"):
            call()


@built
@pytest.mark.parametrize("seqs,length,heads,dim,state", [(2048, 128, 8, 64, 64), (8192, 128, 8, 64, 64), (2048, 512, 32, 64, 128),
                                                         (1, 65536, 16, 64, 128), (300, 509, 8, 64, 64)])
def test_scratch_memory_of_cut_sequences_goes_by_rows_not_by_sequences(seqs, length, heads, dim, state):
    """Scratch memory for states is that of pieces after a sequence's first: a place for each piece's rows of the
    call, however many sequences there are, and in a gradient a state for each 64 rows and the sums of B's and C's."""
    L, rows, inner = trunk.lib(), seqs * length, heads * dim
    a = trunk.CScan(dtype=0, tokens=rows, seqs=seqs, heads=heads, groups=1, dim=dim, state=state, x_stride=inner, y_stride=inner,
                    dt_stride=heads, b_stride=state, c_stride=state, x=16, dt=16, B=16, C=16, A=16, offsets=16)
    one = heads * (dim * state * 4 + 8)  # a piece's states and decays
    order = (rows // 64 + seqs + 2) * 8
    # Pieces are as long as an even share of 4,096 wavefronts, and of at least 64 rows.
    even = -(-rows * heads * (dim // 32) // 4096)
    places = rows // max(64, even) + 1
    assert 0 < L.uor_trunk_scan_workspace_bytes(C.byref(a)) <= places * one + order + 256
    # dA, dD and ddt_bias of each piece; B's and C's gradients in f32 for each of a group's up to 4 x heads wavefronts' turns.
    sums, kept = (places + seqs) * heads * 24, (rows // 64 + 1) * heads * dim * state * 4
    parts = max(1, min(-(-512 // seqs), heads))
    assert L.uor_trunk_scan_backward_workspace_bytes(C.byref(a)) <= 2 * places * one + kept + sums + order + 2 * parts * rows * state * 4 + 4096


def test_a_reply_to_nothing_is_refused():
    """An empty prompt has no last row: its reply would go on from another prompt's."""
    from uor_fbs import float_trunk as ft
    cfg = ft.Config(vocab=8, width=8, layers=1, heads=1, dim=4, state=4)
    p, state = ft.make_params(cfg, device="cpu"), ft.make_state(cfg, 2, device="cpu")
    for offsets in ([0, 3, 3], [0, 0, 3]):
        with pytest.raises(ValueError, match="no tokens"):
            ft.reply(cfg, p, torch.zeros(3, dtype=torch.long), torch.tensor(offsets, dtype=torch.int32), 2, state, torch.tensor([0, 1], dtype=torch.int32))
