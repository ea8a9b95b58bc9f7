"""GPU tests of the float trunk's operators (uor_fbs.trunk) at the edges of what a call may hold: rows that
no sequence owns, offsets of any content, far slots, pieces of several chunks, values that are not finite. Tolerances are
those of the operators' own tests."""

import pytest
import torch

import trunk_cases as oracle
from test_hip_trunk import CONV_UNIT, check_scan, check_scan_backward, conv_case, dtype, near, scan_case, trunk, unit_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def stale(monkeypatch):
    """Memory that a call takes holds NaN, as it may after other work."""
    def filled(make):
        def made(*args, **kw):
            t = make(*args, **kw)
            if t.is_cuda and t.numel():
                t.view(torch.uint8).fill_(255)
            return t
        return made

    monkeypatch.setattr(torch, "empty", filled(torch.empty))
    monkeypatch.setattr(torch, "empty_like", filled(torch.empty_like))


# ---------------------------------------------------------------------------------------------
# Rows that no sequence owns.


def without_ends(x, lengths):
    """The case with its first and last sequence's rows left to nobody."""
    x = {**x, "offsets": oracle.offsets_of(lengths)[1:-1].contiguous().cuda()}
    if x["initial"] is not None:
        x["initial"] = x["initial"][1:-1].contiguous()
    return x


PADDED = [
    # lengths, heads, groups, dim, state; the first and the last are nobody's
    ([3, 37, 0, 26, 14], 2, 1, 32, 16),
    ([70, 20, 5, 90], 8, 1, 32, 20),       # a group's heads in two blocks
    ([9, 1100, 130, 700], 2, 1, 16, 16),   # cut into pieces
    ([5, 0, 0, 0, 200], 3, 3, 65, 33),     # nothing owned at all
]


@pytest.mark.parametrize("shape", PADDED, ids=str)
def test_rows_of_no_sequence_are_zeros(shape, dtype, stale):
    x, m = scan_case(dtype, *shape, initial=True, seed=12)
    x = without_ends(x, shape[0])
    a, b = int(x["offsets"][0]), int(x["offsets"][-1])
    x["x"][:a], x["x"][b:] = 0, 0  # the oracle's dD takes in all rows
    check_scan(x, dtype)
    check_scan_backward(x, m, dtype)
    dy = m(*x["x"].shape)
    want = (*trunk.scan(**x), *trunk.scan_backward(dy, **x))
    assert not any(t[:a].any() or t[b:].any() for t in (want[0], *(want[2 + i] for i in (0, 1, 3, 4))))
    for t in (dy, *(x[k] for k in ("x", "dt", "B", "C"))):
        t[:a], t[b:] = float("nan"), float("nan")
    for one, two in zip(want, (*trunk.scan(**x), *trunk.scan_backward(dy, **x))):
        assert torch.equal(one, two)


@pytest.mark.parametrize("lengths,channels", [([3, 40, 0, 1, 33, 50], 24), ([30, 0, 64], 13), ([1, 700, 900], 8)], ids=str)
def test_rows_of_no_sequence_are_zeros_in_the_convolution(lengths, channels, dtype, stale):
    x, m = conv_case(dtype, lengths, channels, 4, True, seed=3)
    x = without_ends(x, lengths)
    y, final = trunk.conv(**x)
    want, last, size = oracle.conv(**x)
    near("y", y, want, size * 1.1, dtype, CONV_UNIT)
    assert torch.equal(final.cpu().double(), last)
    dy, dfinal = m(*y.shape), m(*final.shape)
    got = trunk.conv_backward(dy, **x, dfinal=dfinal)
    grads, sizes = oracle.conv_backward(dy, **x, dfinal=dfinal)
    for name in trunk.ConvGrads._fields:
        near(name, getattr(got, name), grads[name], sizes[name], torch.float32 if name in ("dweight", "dbias") else dtype,
             CONV_UNIT + (sum(lengths) * 2.0 ** -24 if name in ("dweight", "dbias") else 0))
    a, b = int(x["offsets"][0]), int(x["offsets"][-1])
    for t in (y, got.dx):
        assert not t[:a].any() and not t[b:].any()


# ---------------------------------------------------------------------------------------------
# Places.


@pytest.mark.parametrize("far", [1 << 32, (1 << 32) + 1, 1 << 31, -(1 << 32) + 1, 1 << 62])
def test_slots_past_32_bits_are_skipped(far, dtype):
    x, m = scan_case(dtype, [3], 2, 1, 16, 16)
    states = m.f32(4, 2, 16, 16)
    kept = states.clone()
    slots = torch.tensor([3, far, 2]).cuda()
    y = trunk.scan_step(**{k: x[k] for k in ("x", "dt", "A", "B", "C")}, states=states, slots=slots)
    assert not y[1].any() and y[0].any() and y[2].any()
    assert torch.equal(states[:2], kept[:2]) and not torch.equal(states[2:], kept[2:])
    c, m = conv_case(dtype, [3], 8, 4, False)
    held = m(4, 3, 8)
    kept = held.clone()
    y = trunk.conv_step(c["x"], c["weight"], held, slots=slots)
    assert not y[1].any() and torch.equal(held[:2], kept[:2]) and not torch.equal(held[2:], kept[2:])


def test_offsets_past_32_bits_are_the_nearest_inside(dtype):
    x, m = scan_case(dtype, [40, 60], 2, 1, 32, 32)
    dy = m(*x["x"].shape)
    want = (*trunk.scan(**x), *trunk.scan_backward(dy, **x)[:7])
    x["offsets"] = torch.tensor([-(1 << 32) + 7, 40, (1 << 32) + 50]).cuda()
    for a, b in zip(want, (*trunk.scan(**x), *trunk.scan_backward(dy, **x)[:7])):
        assert torch.equal(a, b)
    c, _ = conv_case(dtype, [40, 60], 16, 4, False)
    want = trunk.conv(**c)
    c["offsets"] = x["offsets"]
    for a, b in zip(want, trunk.conv(**c)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("stride", [0, 8, -64])
def test_one_row_has_no_stride(stride, dtype):
    """From C: the strides of a call of one row are not looked at."""
    x, m = scan_case(dtype, [1], 2, 1, 64, 64, initial=True)
    dy, df = m(*x["x"].shape), m.f32(1, 2, 64, 64)
    y, final = trunk.scan(**x)
    grads = trunk.scan_backward(dy, **x, dfinal=df)
    a, keep = trunk._scan_args(*(x[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "offsets", "initial")))
    a.x_stride = a.dt_stride = a.b_stride = a.c_stride = a.y_stride = stride
    y2, final2 = torch.empty_like(y), torch.empty_like(final)
    a.y, a.final = y2.data_ptr(), final2.data_ptr()
    trunk._call("scan", a, 0)
    assert torch.equal(y, y2) and torch.equal(final, final2)
    got = trunk.ScanGrads(*(torch.empty_like(g) for g in grads))
    a.dy, a.dfinal = dy.data_ptr(), df.data_ptr()
    a.dx, a.ddt, a.dA, a.dB, a.dC, a.dD, a.ddt_bias, a.dinitial = (g.data_ptr() for g in got)
    trunk._call("scan_backward", a, 0)
    for one, two in zip(grads, got):
        assert torch.equal(one, two)


# ---------------------------------------------------------------------------------------------
# Gradients of pieces of several chunks: states kept between them, the walk along a piece and back.


LONG = [
    # lengths, heads, groups, dim, state, chunks that the longest piece has
    ([450, 449, 320, 193, 192, 129, 128, 65, 64, 63, 0, 1, 130] + [45] * 64, 16, 2, 40, 72, 3),
    ([1300, 640, 641, 577, 576, 449, 193, 129, 128, 0, 1] + [130] * 38, 64, 8, 8, 16, 9),
    ([250, 0, 193] + [37] * 125, 16, 16, 5, 33, 1),
]


def kept_bytes(x):
    """What the states of all chunks take in a gradient's scratch memory."""
    rows, heads, dim = x["x"].shape
    state = x["B"].shape[2]
    parts, padded = (1 if dim <= 32 else 2 if dim <= 64 else 4), (32 if state <= 32 else 64 if state <= 64 else 128)
    return (rows // 64 + 1) * heads * parts * padded * 32 * 4


@pytest.mark.parametrize("shape", LONG, ids=["3 chunks, state 72", "9 chunks", "64 rows, a group a head"])
def test_scan_backward_of_pieces_of_several_chunks(shape, dtype):
    lengths, heads, groups, dim, state, chunks = shape
    x, m = scan_case(dtype, lengths, heads, groups, dim, state, initial=True, seed=21)
    rows, units = sum(lengths), heads * (1 if dim <= 32 else 2)
    assert len(lengths) * units >= 2048  # sequences enough that only those far over an even share are cut
    assert -(-4 * -(-rows * units // 4096) // 64) >= chunks
    args, _ = trunk._scan_args(*(x[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "offsets", "initial")))
    got = trunk.lib().uor_trunk_scan_backward_workspace_bytes(args)
    if chunks >= 9:
        assert got >= kept_bytes(x)  # more than all else together: pieces are of three chunks or more
    check_scan(x, dtype)
    check_scan_backward(x, m, dtype)


# ---------------------------------------------------------------------------------------------
# Values that are not finite: by the definition they reach some results, and no others.


def same_where_finite(name, got, want, size, dtype, unit):
    """got is finite exactly where the definition is, and near it there."""
    there = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got).cpu(), there), (name, int((torch.isfinite(got).cpu() != there).sum()), int((~there).sum()))
    near(name, got.cpu()[there], want[there], size[there], dtype, unit)


def check_odd(x, dy, df, dtype):
    dim, state = x["x"].shape[2], x["B"].shape[2]
    unit = unit_of(dtype, 64 + state + 32)
    for name, got, want, size in zip(("y", "final"), trunk.scan(**x), oracle.scan(**x), oracle.scan(**x, magnitude=True)):
        same_where_finite(name, got, want, size, dtype if name == "y" else torch.float32, unit)
    got = trunk.scan_backward(dy, **x, dfinal=df)
    want = oracle.scan_backward(dy, **x, dfinal=df)
    size = oracle.scan_backward(dy, **x, dfinal=df, magnitude=True)
    unit = unit_of(dtype, 2 * (64 + dim + state + 32))
    a = x["A"].cpu().double().abs()
    later = torch.zeros_like(size["q"])
    for s, e in oracle.bounds(x["offsets"], x["x"].shape[0]):
        for t in range(s, e):
            later[t] = torch.nan_to_num(size["q"][t:min(e, t + 64)], nan=0.0, posinf=0.0).sum(0)
    size["ddt"] = size["ddt"] + a * later
    size["dA"] = size["dA"] + (size["step"] * later).sum(0)
    size["ddt_bias"] = size["ddt_bias"] + (a * later).sum(0)
    for name in trunk.ScanGrads._fields:
        if want[name] is None:
            assert getattr(got, name) is None
            continue
        kind = dtype if name in ("dx", "ddt", "dB", "dC") else torch.float32
        same_where_finite(name, getattr(got, name), want[name], size[name], kind, unit + (0 if kind == dtype == torch.bfloat16 else 64 * 2.0 ** -24))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", ["x", "dt", "B", "C", "dy", "initial", "dfinal", "A", "D", "dt_bias"])
def test_what_is_not_finite_reaches_what_depends_on_it(name, value, dtype):
    """One value of each input, at the ends and in the middle of chunks and of their tiles; the sequence
    before and the one after, the other head and the other group have none."""
    x, m = scan_case(dtype, [30, 150, 40], 4, 2, 40, 20, initial=True, seed=31)
    dy, df = m(*x["x"].shape), m.f32(3, 4, 40, 20)
    rows = [30 + t for t in (0, 5, 37, 63, 64, 100, 149)]
    for row in rows if name in ("x", "dt", "B", "C", "dy") else [1]:
        bad = {**x, "dy": dy, "dfinal": df}
        t = bad[name] = bad[name].clone()
        place = (row, 2, 7, 11)[:t.dim()] if t.dim() > 1 else (2,)
        if name in ("B", "C"):
            place = (row, 1, 7)
        t[place] = value
        if name == "A":
            t[2] = -abs(value)
        check_odd({k: v for k, v in bad.items() if k not in ("dy", "dfinal")}, bad["dy"], bad["dfinal"], dtype)


@pytest.mark.parametrize("name", ["x", "dt", "B", "C", "dy"])
def test_what_is_not_finite_in_long_and_cut_sequences(name, dtype):
    """Several odd rows, in sequences of several pieces, and without states before and after."""
    x, m = scan_case(dtype, [3, 700, 64], 8, 1, 32, 33, seed=32)
    dy = m(*x["x"].shape)
    bad = {**x, "dy": dy}
    t = bad[name] = bad[name].clone()
    for row, value in ((3 + 200, float("nan")), (3 + 201, float("inf")), (3 + 333, -float("inf")), (3 + 699, float("nan"))):
        t[(row, 0, 3)[:t.dim()] if name != "dt" else (row, 5)] = value
    dy = bad.pop("dy")
    check_odd(bad, dy, None, dtype)


@pytest.mark.parametrize("name", ["x", "dt", "B", "C", "dy"])
def test_what_is_not_finite_in_pieces_of_several_chunks(name, dtype):
    x, m = scan_case(dtype, [450, 320, 130] + [60] * 32, 64, 8, 8, 16, initial=True, seed=33)
    dy, df = m(*x["x"].shape), m.f32(35, 64, 8, 16)
    assert 35 * 64 >= 2048 and -(-4 * -(-x["x"].shape[0] * 64 // 4096) // 64) >= 3
    bad = {**x, "dy": dy}
    t = bad[name] = bad[name].clone()
    for row in (70, 450 + 200, 450 + 320 + 129):
        t[(row, 1, 3)[:t.dim()]] = float("nan")
    dy = bad.pop("dy")
    check_odd(bad, dy, df, dtype)


# ---------------------------------------------------------------------------------------------
# Offsets that do not ascend: no promise is made of the results, but nothing outside the arrays is written.


@pytest.fixture
def fenced(monkeypatch):
    """Everything that a call allocates lies between two stretches of 64 KB that stay as they are."""
    fences, edge, make = [], 1 << 16, torch.empty

    def fence(shape, dtype, device):
        shape = tuple(shape) if isinstance(shape, (tuple, list, torch.Size)) else (shape,)
        size = 1
        for s in shape:
            size *= s
        n = size * dtype.itemsize
        whole = make(2 * edge + (n + 255) // 256 * 256, dtype=torch.uint8, device=device).fill_(0x5a)
        fences.append((whole, n))
        return whole[edge:edge + n].view(dtype).view(shape)

    monkeypatch.setattr(torch, "empty", lambda *shape, dtype, device: fence(shape[0] if len(shape) == 1 else shape, dtype, device))
    monkeypatch.setattr(torch, "empty_like", lambda t, memory_format=None: fence(t.shape, t.dtype, t.device))
    yield lambda: [w for w, n in fences if bool((w[:edge] != 0x5a).any()) or bool((w[edge + n:] != 0x5a).any())]


@pytest.mark.parametrize("rows", [130, 1500])
@pytest.mark.parametrize("offsets", [[0, 50, 20, 90, 10, 130], [130, 0, 130, 0], [1 << 30, -7, 60, -(1 << 31), 1400], [90, 90, 10], [700, 0, 1500, 600, 1500]],
                         ids=str)
def test_offsets_that_do_not_ascend_write_nothing_outside(offsets, rows, dtype, fenced):
    x, m = scan_case(dtype, [rows], 4, 2, 40, 20)
    n = len(offsets) - 1
    x["offsets"] = torch.tensor(offsets, dtype=torch.int32).cuda()
    x["initial"] = m.f32(n, 4, 40, 20)
    c, _ = conv_case(dtype, [rows], 24, 4, False)
    c.update(offsets=x["offsets"], initial=m(n, 3, 24))
    dy, df, dyc, dfc = m(rows, 4, 40), m.f32(n, 4, 40, 20), m(rows, 24), m(n, 3, 24)
    kept = {k: v.clone() for k, v in (*x.items(), *((f"conv {k}", v) for k, v in c.items()))}
    trunk.scan(**x)
    trunk.scan_backward(dy, **x, dfinal=df)
    trunk.conv(**c)
    trunk.conv_backward(dyc, **c, dfinal=dfc)
    torch.cuda.synchronize()
    assert not fenced()
    for k, v in kept.items():
        assert torch.equal(v, c[k[5:]] if k.startswith("conv ") else x[k])
    # And the next call is as any other.
    x["offsets"], x["initial"] = oracle.offsets_of([rows]).cuda(), None
    check_scan(x, dtype)
