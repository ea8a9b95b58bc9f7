"""GPU tests of the float trunk's operators (uor_fbs.trunk) against their definitions in 64 bits.

Tolerances. An output's own rounding is half a step of its type, `eps / 2` of its value. Before it
stand sums in 32 bits. An f32 call's products and sums are each off by 2^-24 of the sum of absolute
terms, once a term: a row's sums have at most chunk + state + dim terms here, and a decay, the
exponential of a sum of logarithms whose parts are good to their own size, counts as 16 terms; a
gradient goes through two such sums. A bf16 call's operands that were computed in 32 bits are two
bf16 parts, each product off by 2^-18 of its size; two such in a row and the sums in 32 bits stay
under 2^-16. Sums over all rows (the parameters' gradients) add 2^-24 for each of 64 terms, as they
go over rows in chunks. The state's axis enters through `magnitude`, the same sums over absolute
values, which each error is relative to.
"""

import pytest
import torch

import trunk_cases as oracle

pytestmark = pytest.mark.gpu
trunk = pytest.importorskip("uor_fbs.trunk")

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(params=list(TYPES))
def dtype(request):
    return TYPES[request.param]


class Make:
    def __init__(self, dtype, seed):
        self.dtype, self.gen = dtype, torch.Generator().manual_seed(seed)

    def __call__(self, *shape, scale=1.0):
        return (torch.randn(shape, generator=self.gen) * scale).to(self.dtype).cuda()

    def f32(self, *shape, scale=1.0, mean=0.0):
        return (torch.randn(shape, generator=self.gen) * scale + mean).cuda()


def near(name, got, want, size, dtype, unit):
    """got within its type's half step of want and `unit` of the sums' size."""
    assert got.dtype == dtype, name
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    allowed = torch.finfo(dtype).eps / 2 * want.abs() + unit * size * (1 + torch.finfo(dtype).eps) + 1e-30
    off = (got - want).abs()
    bad = ~(off <= allowed)
    assert not bad.any(), (name, int(bad.sum()), float(off[bad].max()), float((off / allowed)[bad].max()))


def unit_of(dtype, terms):
    return 2.0 ** -16 if dtype == torch.bfloat16 else terms * 2.0 ** -24


def scan_case(dtype, lengths, heads, groups, dim, state, initial=False, seed=1, step=0.0):
    m = Make(dtype, seed)
    rows = sum(lengths)
    x = dict(x=m(rows, heads, dim), dt=m(rows, heads, scale=0.7), A=-m.f32(heads).abs() - 0.05, B=m(rows, groups, state, scale=0.5),
             C=m(rows, groups, state, scale=0.5), D=m.f32(heads), dt_bias=m.f32(heads, scale=0.5, mean=step - 1.0),
             offsets=oracle.offsets_of(lengths).cuda(),
             initial=m.f32(len(lengths), heads, dim, state) if initial else None)
    return x, m


def check_scan(x, dtype):
    y, final = trunk.scan(**x)
    want, last = oracle.scan(**x)
    size, size_last = oracle.scan(**x, magnitude=True)
    terms = 64 + x["B"].shape[2] + 32
    near("y", y, want, size, dtype, unit_of(dtype, terms))
    near("final", final, last, size_last, torch.float32, unit_of(dtype, terms))
    return y, final


SHAPES = [
    # lengths, heads, groups, dim, state
    ([1], 1, 1, 1, 1),
    ([64], 2, 1, 64, 64),
    ([65, 63, 1], 4, 2, 64, 32),
    ([0, 130, 0, 17, 128], 3, 3, 16, 20),
    ([77], 6, 2, 40, 128),
    ([33, 100], 2, 1, 128, 48),
    ([5, 0, 0, 70], 2, 2, 65, 33),
    ([200, 3], 1, 1, 31, 127),
]


@pytest.mark.parametrize("initial", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan(shape, initial, dtype):
    x, _ = scan_case(dtype, *shape, initial=initial)
    check_scan(x, dtype)


def test_scan_without_the_parameters_that_may_be_absent(dtype):
    x, _ = scan_case(dtype, [70, 9], 2, 1, 32, 16)
    x.update(D=None, dt_bias=None)
    check_scan(x, dtype)
    one, _ = scan_case(dtype, [90], 2, 1, 32, 16)
    one["offsets"] = None
    check_scan(one, dtype)


def test_scan_cut_into_pieces(dtype):
    """Sequences long enough to be cut, ends inside a piece, at its end and after many pieces."""
    x, _ = scan_case(dtype, [1100, 0, 256, 7, 513], 2, 1, 32, 16, initial=True, seed=5)
    check_scan(x, dtype)


def test_scan_goes_on_from_its_final_state(dtype):
    x, _ = scan_case(dtype, [150], 4, 2, 64, 64, seed=8)
    y, final = trunk.scan(**x)
    cut = lambda a, b: {**x, **{k: x[k][a:b] for k in ("x", "dt", "B", "C")}, "offsets": None}  # noqa: E731
    first, held = trunk.scan(**cut(0, 90))
    second, end = trunk.scan(**{**cut(90, 150), "initial": held})
    size, size_last = oracle.scan(**x, magnitude=True)
    unit = 2 * unit_of(dtype, 64 + 64 + 32)
    near("y", torch.cat([first, second]), y.cpu().double(), size + y.cpu().double().abs() * 2 ** 8 * (dtype == torch.bfloat16), dtype, unit)
    near("final", end, final.cpu().double(), size_last, torch.float32, unit)


def test_scan_of_long_steps(dtype):
    """Decays that leave nothing: sums of logarithms far past the exponents' range."""
    x, _ = scan_case(dtype, [140, 64], 2, 1, 32, 32, initial=True, step=400.0)
    check_scan(x, dtype)


def test_scan_of_strided_and_unaligned_rows(dtype):
    x, m = scan_case(dtype, [70, 60], 4, 2, 24, 16)
    want = trunk.scan(**x)
    wide = m(130, 4 * 24 + 2 * 2 * 16 + 4 + 3)
    rows = wide[:, 1:]
    cols = [4 * 24, 2 * 16, 2 * 16, 4]
    at, parts = 0, []
    for c, t in zip(cols, (x["x"], x["B"], x["C"], x["dt"])):
        part = rows[:, at:at + c].unflatten(1, t.shape[1:])
        part.copy_(t)
        parts.append(part)
        at += c
    assert not parts[0].is_contiguous()
    got = trunk.scan(**{**x, "x": parts[0], "B": parts[1], "C": parts[2], "dt": parts[3]})
    turned = x["x"].transpose(1, 2).contiguous().transpose(1, 2)
    again = trunk.scan(**{**x, "x": turned})
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", ["x", "dt", "B", "C"])
def test_what_comes_later_reaches_no_row_before(name, value, dtype):
    x, _ = scan_case(dtype, [100, 50], 2, 1, 64, 32)
    want, last = trunk.scan(**x)
    for row in (0, 37, 64, 99):
        bad = {**x, name: x[name].clone()}
        bad[name][row] = value
        y, final = trunk.scan(**bad)
        near("before", y[:row], want[:row].cpu().double(), torch.zeros(1), dtype, 0)
        near("the other", y[100:], want[100:].cpu().double(), torch.zeros(1), dtype, 0)
        near("its state", final[1:], last[1:].cpu().double(), torch.zeros(1), torch.float32, 0)
        if value != value:
            assert not torch.isfinite(y[row].float()).any()


def test_calls_give_the_same_bits_each_time_and_on_another_stream(dtype):
    x, m = scan_case(dtype, [700, 64, 300], 4, 2, 64, 64)
    dy = m(*x["x"].shape)
    want = (*trunk.scan(**x), *trunk.scan_backward(dy, **x)[:7])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = (*trunk.scan(**x), *trunk.scan_backward(dy, **x)[:7])
    stream.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_offsets_of_any_content_stay_inside_the_rows(dtype):
    """Offsets are clamped; the sequences that ascend are right all the same."""
    x, _ = scan_case(dtype, [40, 60], 2, 1, 32, 32)
    y, final = trunk.scan(**x)
    x["offsets"] = torch.tensor([-5, 40, 1 << 30], dtype=torch.int32).cuda()
    got = trunk.scan(**x)
    assert torch.equal(got[0], y) and torch.equal(got[1], final)


# ---------------------------------------------------------------------------------------------
# The scan's gradients.


def check_scan_backward(x, m, dtype, dfinal=True):
    dy = m(*x["x"].shape)
    seqs = 1 if x["offsets"] is None else x["offsets"].numel() - 1
    heads, dim, state = x["x"].shape[1], x["x"].shape[2], x["B"].shape[2]
    df = m.f32(seqs, heads, dim, state) if dfinal else None
    got = trunk.scan_backward(dy, **x, dfinal=df)
    want = oracle.scan_backward(dy, **x, dfinal=df)
    size = oracle.scan_backward(dy, **x, dfinal=df, magnitude=True)
    # A row's da is a sum over the rows that follow it in its chunk, less what they have of their own.
    for a, b in oracle.bounds(x["offsets"], x["x"].shape[0]):
        for t in range(a, b):
            later = size["q"][t:min(b, t + 64)].sum(0)
            size["ddt"][t] += x["A"].cpu().double().abs() * later
            size["dA"] += size["step"][t] * later
            if size["ddt_bias"] is not None:
                size["ddt_bias"] += x["A"].cpu().double().abs() * later
    unit = unit_of(dtype, 2 * (64 + dim + state + 32))
    for name in trunk.ScanGrads._fields:
        g = getattr(got, name)
        if want[name] is None:
            assert g is None
            continue
        kind = dtype if name in ("dx", "ddt", "dB", "dC") else torch.float32
        near(name, g, want[name], size[name], kind, unit + (0 if kind == dtype == torch.bfloat16 else 64 * 2.0 ** -24))
    return got


@pytest.mark.parametrize("initial", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan_backward(shape, initial, dtype):
    x, m = scan_case(dtype, *shape, initial=initial, seed=2)
    check_scan_backward(x, m, dtype, dfinal=initial)


def test_scan_backward_cut_into_pieces(dtype):
    x, m = scan_case(dtype, [1100, 0, 256, 7, 513], 2, 1, 32, 16, initial=True, seed=6)
    check_scan_backward(x, m, dtype)


def test_scan_backward_of_long_steps_and_absent_parameters(dtype):
    x, m = scan_case(dtype, [140, 64], 2, 1, 32, 32, step=400.0)
    check_scan_backward(x, m, dtype)
    x, m = scan_case(dtype, [90], 4, 1, 32, 16)
    x.update(D=None, dt_bias=None, offsets=None)
    check_scan_backward(x, m, dtype)


def test_scan_backward_of_many_heads_a_group(dtype):
    x, m = scan_case(dtype, [30, 40], 12, 2, 16, 16)
    check_scan_backward(x, m, dtype)


# ---------------------------------------------------------------------------------------------
# Single tokens.


@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (9, 4, 2, 64, 64), (3, 6, 3, 33, 20), (5, 2, 1, 128, 128), (2, 2, 2, 7, 50)], ids=str)
def test_scan_step(shape, dtype):
    rows, heads, groups, dim, state = shape
    x, m = scan_case(dtype, [rows], heads, groups, dim, state)
    x = {k: x[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias")}
    states = m.f32(rows + 3, heads, dim, state)
    index = torch.randperm(rows + 3, generator=m.gen)[:rows].int()
    if rows > 2:
        index[1], index[2] = -1, rows + 3  # skipped
    want, held = oracle.scan_step(**x, states=states, index=index)
    size, size_held = oracle.scan_step(**x, states=states, index=index, magnitude=True)
    y = trunk.scan_step(**x, states=states, slots=index.cuda())
    unit = (state + 16) * 2.0 ** -24
    near("y", y, want, size, dtype, unit)
    near("states", states, held, size_held, torch.float32, unit)


def test_steps_follow_the_scan(dtype):
    x, _ = scan_case(dtype, [20], 4, 2, 32, 32)
    y, final = trunk.scan(**x)
    states = torch.zeros_like(final)
    got = [trunk.scan_step(**{k: x[k][t:t + 1] for k in ("x", "dt", "B", "C")}, states=states, **{k: x[k] for k in ("A", "D", "dt_bias")})
           for t in range(20)]
    size, size_last = oracle.scan(**x, magnitude=True)
    unit = 2 * unit_of(dtype, 64 + 32 + 32) + 20 * 2.0 ** -24
    near("y", torch.cat(got), y.cpu().double(), size + y.cpu().double().abs() * 2 ** 8 * (dtype == torch.bfloat16), dtype, unit)
    near("state", states, final.cpu().double(), size_last, torch.float32, unit)


# ---------------------------------------------------------------------------------------------
# The convolution. Its sums have taps + 1 terms, and silu six more roundings.


CONV_UNIT = 16 * 2.0 ** -24


def conv_case(dtype, lengths, channels, taps, initial, seed=1):
    m = Make(dtype, seed)
    return dict(x=m(sum(lengths), channels), weight=m.f32(channels, taps), bias=m.f32(channels), offsets=oracle.offsets_of(lengths).cuda(),
                initial=m(len(lengths), taps - 1, channels) if initial else None), m


CONVS = [([1], 1), ([40, 0, 2, 1, 33], 8), ([100, 3], 24), ([64, 32, 31], 13), ([7], 520)]


@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("taps", [1, 2, 3, 4])
@pytest.mark.parametrize("lengths,channels", CONVS, ids=str)
def test_conv(lengths, channels, taps, silu, dtype):
    x, m = conv_case(dtype, lengths, channels, taps, initial=silu)
    y, final = trunk.conv(**x, silu=silu)
    want, last, size = oracle.conv(**x, silu=silu)
    near("y", y, want, size * 1.1, dtype, CONV_UNIT)  # silu's slope is below 1.1
    assert torch.equal(final.cpu().double(), last)
    dy, dfinal = m(*y.shape), m(*final.shape) if silu else None
    got = trunk.conv_backward(dy, **x, dfinal=dfinal, silu=silu)
    grads, sizes = oracle.conv_backward(dy, **x, dfinal=dfinal, silu=silu)
    for name in trunk.ConvGrads._fields:
        if name == "dinitial" and not silu:
            assert got.dinitial is None
            continue
        near(name, getattr(got, name), grads[name], sizes[name], torch.float32 if name in ("dweight", "dbias") else dtype,
             CONV_UNIT + (sum(lengths) * 2.0 ** -24 if name in ("dweight", "dbias") else 0))


def test_conv_of_strided_rows_and_no_bias(dtype):
    x, m = conv_case(dtype, [50, 20], 24, 4, False)
    x["bias"] = None
    y, _ = trunk.conv(**x)
    for lead in (1, 8):
        wide = m(70, 24 + 16)
        part = wide[:, lead:lead + 24]
        part.copy_(x["x"])
        got, _ = trunk.conv(**{**x, "x": part})
        assert torch.equal(got, y)
        dy = m(*y.shape)
        for a, b in zip(trunk.conv_backward(dy, **x), trunk.conv_backward(dy, **{**x, "x": part})):
            assert a is None and b is None or torch.equal(a, b)


@pytest.mark.parametrize("taps", [1, 2, 4])
def test_conv_steps_follow_the_convolution(taps, dtype):
    x, m = conv_case(dtype, [9, 9, 9], 21, taps, True)
    y, final = trunk.conv(**x)
    states = m(6, taps - 1, 21)
    others = states.clone()
    slots = torch.tensor([4, 0, 3], dtype=torch.int32).cuda()
    states[slots.long()] = x["initial"]
    rows = x["x"].view(3, 9, 21)
    for t in range(9):
        got = trunk.conv_step(rows[:, t].contiguous(), x["weight"], states, x["bias"], slots=slots)
        assert torch.equal(got, y.view(3, 9, 21)[:, t])
    assert torch.equal(states[slots.long()], final) and torch.equal(states[[1, 2, 5]], others[[1, 2, 5]])
    kept = states.clone()
    got = trunk.conv_step(rows[:2, 0].contiguous(), x["weight"], states, x["bias"], slots=torch.tensor([-1, 6]).cuda())
    assert torch.equal(states, kept) and not got.any()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_conv_reaches_no_row_before_nor_another_sequence(value, dtype):
    x, _ = conv_case(dtype, [10, 10], 16, 4, False)
    y, _ = trunk.conv(**x)
    x["x"][9] = value
    got, _ = trunk.conv(**x)
    assert torch.equal(got[:9], y[:9]) and torch.equal(got[10:], y[10:])


# ---------------------------------------------------------------------------------------------
# The norms: each output goes through at most two sums over the width and twelve roundings a value.


NORMS = [(1, 1), (3, 8), (5, 13), (70, 64), (9, 256), (4, 500), (3, 520), (6, 1000), (2, 1032), (3, 4096), (2, 4100), (1, 8192)]


def norm_unit(width):
    return (24 + 2 * min(width, 64)) * 2.0 ** -24


@pytest.mark.parametrize("absent", [(), ("gate",), ("residual",), ("out", "gate", "post", "scale"), ("pre",), ("post", "scale")], ids=str)
@pytest.mark.parametrize("rows,width", NORMS, ids=str)
def test_norms(rows, width, absent, dtype):
    m = Make(dtype, rows + width)
    x = dict(residual=m(rows, width, scale=2.0), out=m(rows, width), gate=m(rows, width), post=m.f32(width, scale=0.3, mean=1.0),
             scale=m.f32(width), pre=m.f32(width, scale=0.3, mean=1.0))
    x = {k: None if k in absent else v for k, v in x.items()}
    unit = norm_unit(width)
    r, n = trunk.norms(**x)
    want_r, want_n = oracle.norms(**x)
    block = oracle.norms(None, x["out"], x["gate"], x["post"], x["scale"])[0].abs() if x["out"] is not None else 0
    size = block + (0 if x["residual"] is None else x["residual"].cpu().double().abs())
    if x["out"] is None:
        assert r is x["residual"]
    else:
        near("residual", r, want_r, size, dtype, unit)
    if x["pre"] is None:
        assert n is None
    else:
        inverse = 1 / torch.sqrt((want_r * want_r).mean(-1, keepdim=True) + 1e-6)
        # The mean of squares moves with all of the row's errors.
        near("normed", n, want_n, (size + want_r.abs() * (size * want_r.abs()).mean(-1, keepdim=True) * inverse ** 2)
             * inverse * x["pre"].cpu().double().abs(), dtype, unit)


@pytest.mark.parametrize("absent", [(), ("gate",), ("residual",), ("out", "gate", "post", "scale"), ("pre",), ("post", "scale")], ids=str)
@pytest.mark.parametrize("rows,width", NORMS[1:], ids=str)
def test_norms_backward(rows, width, absent, dtype):
    m = Make(dtype, rows + width)
    x = dict(residual=m(rows, width, scale=4.0), out=m(rows, width), gate=m(rows, width), post=m.f32(width, scale=0.3, mean=1.0),
             scale=m.f32(width, scale=0.3), pre=m.f32(width, scale=0.3, mean=1.0))
    x = {k: None if k in absent else v for k, v in x.items()}
    dr, dn = m(rows, width), None if x["pre"] is None else m(rows, width)
    got = trunk.norms_backward(dr, dn, **x)
    want, size = oracle.norms_backward(dr, dn, **x)
    # The residual's own errors move its norm's gradient in proportion, as do the norms' means: each
    # value's error is bounded by its row's largest size.
    for name in trunk.NormGrads._fields:
        if want[name] is None:
            assert getattr(got, name) is None, name
            continue
        rowwise = name in ("dresidual", "dout", "dgate")
        allowed = size[name] + (size[name].amax(-1, keepdim=True) if rowwise else 0)
        near(name, getattr(got, name), want[name], allowed, dtype if rowwise else torch.float32,
             4 * norm_unit(width) + (0 if rowwise else rows * 2.0 ** -24))


def test_norms_of_many_and_strided_rows(dtype):
    m = Make(dtype, 3)
    x = dict(residual=m(9000, 64), out=m(9000, 64), gate=m(9000, 64), post=m.f32(64), scale=m.f32(64), pre=m.f32(64))
    r, n = trunk.norms(**x)
    want_r, want_n = oracle.norms(**x)
    size = want_r.abs() + x["residual"].cpu().double().abs() * 2
    near("residual", r, want_r, size, dtype, norm_unit(64))
    wide = m(9000, 3 * 64 + 1)
    parts = [wide[:, 1 + 64 * i:65 + 64 * i] for i in range(3)]
    for p, k in zip(parts, ("residual", "out", "gate")):
        p.copy_(x[k])
    got = trunk.norms(**{**x, "residual": parts[0], "out": parts[1], "gate": parts[2]})
    assert torch.equal(got[0], r) and torch.equal(got[1], n)
    dr, dn = m(9000, 64), m(9000, 64)
    for a, b in zip(trunk.norms_backward(dr, dn, **x),
                    trunk.norms_backward(dr, dn, **{**x, "residual": parts[0], "out": parts[1], "gate": parts[2]})):
        assert torch.equal(a, b)


def test_norms_of_no_rows_and_rows_of_zeros(dtype):
    m = Make(dtype, 3)
    r, n = trunk.norms(m(0, 32), m(0, 32), pre=m.f32(32))
    assert r.shape == n.shape == (0, 32)
    got = trunk.norms_backward(m(0, 32), m(0, 32), m(0, 32), m(0, 32), post=m.f32(32), pre=m.f32(32))
    assert not got.dpost.any() and not got.dpre.any()
    zero = torch.zeros(2, 32, dtype=dtype).cuda()
    r, n = trunk.norms(zero, zero, pre=m.f32(32))
    assert not r.any() and not n.any()


def test_calls_of_no_rows(dtype):
    x, m = scan_case(dtype, [0, 0], 2, 1, 16, 16, initial=True)
    y, final = trunk.scan(**x)
    assert y.shape[0] == 0 and torch.equal(final, x["initial"])
    got = trunk.scan_backward(m(0, 2, 16), **x, dfinal=x["initial"])
    assert torch.equal(got.dinitial, x["initial"]) and not got.dA.any() and not got.dD.any()
    c, m = conv_case(dtype, [0, 0], 16, 4, True)
    y, final = trunk.conv(**c)
    assert torch.equal(final, c["initial"])
    got = trunk.conv_backward(m(0, 16), **c, dfinal=c["initial"])
    assert torch.equal(got.dinitial, c["initial"]) and not got.dweight.any()
    assert trunk.scan_step(**{k: x[k] for k in ("x", "dt", "A", "B", "C")}, states=x["initial"]).shape[0] == 0


@pytest.mark.parametrize("state", [20, 33])
def test_scan_of_many_short_sequences(state, dtype):
    """More sequences than one look of the search takes, and a group's heads in turns of one block."""
    lengths = [(i * 7) % 4 for i in range(600)]
    x, m = scan_case(dtype, lengths, 8, 1, 32, state, initial=True, seed=9)
    check_scan(x, dtype)
    check_scan_backward(x, m, dtype)


def test_scan_of_many_rows_in_order_of_length(dtype):
    """Calls large enough to go through their sequences by length give what smaller ones give."""
    lengths = [(i * 37) % 161 for i in range(450)]
    x, m = scan_case(dtype, lengths, 16, 2, 32, 16, seed=4)
    assert sum(lengths) >= 32768
    dy = m(*x["x"].shape)
    (y, final), grads = trunk.scan(**x), trunk.scan_backward(dy, **x)
    cuts = [0, 200, 450]
    for a, b in zip(cuts, cuts[1:]):
        rows = slice(sum(lengths[:a]), sum(lengths[:b]))
        part = {**x, **{k: x[k][rows] for k in ("x", "dt", "B", "C")}, "offsets": oracle.offsets_of(lengths[a:b]).cuda()}
        y2, final2 = trunk.scan(**part)
        assert torch.equal(y[rows], y2) and torch.equal(final[a:b], final2)
        some = trunk.scan_backward(dy[rows], **part)
        for name in ("dx", "ddt", "dB", "dC"):
            assert torch.equal(getattr(grads, name)[rows], getattr(some, name)), name


def test_scan_of_thousands_of_sequences(dtype):
    x, _ = scan_case(dtype, [1] * 5000, 1, 1, 4, 3, initial=True, seed=3)
    check_scan(x, dtype)


def test_scan_of_rows_far_apart(dtype):
    """Rows whose chunk's offsets pass 31 bits in bytes: read without them."""
    x, m = scan_case(dtype, [3], 2, 1, 16, 16)
    wide = m(3, 1 << 22)
    want = trunk.scan(**x)
    dy = m(*x["x"].shape)
    grads = trunk.scan_backward(dy, **x)
    far = {k: x[k] for k in ("x", "B", "C")}
    at = 8
    for k, t in far.items():
        n = t[0].numel()
        part = wide[:, at:at + n].unflatten(1, t.shape[1:])
        part.copy_(t)
        far[k], at = part, at + n
    assert far["x"].stride(0) == 1 << 22
    for a, b in zip((*want, *grads), (*trunk.scan(**{**x, **far}), *trunk.scan_backward(dy, **{**x, **far}))):
        assert a is None and b is None or torch.equal(a, b)


@pytest.mark.parametrize("channels", [5, 50, 761, 2100])
def test_conv_of_other_numbers_of_channels(channels, dtype):
    """Few channels share a block, many take several; runs end at, before and past a batch's rows."""
    x, m = conv_case(dtype, [33, 0, 64, 1, 31, 70], channels, 3, initial=True, seed=channels)
    y, final = trunk.conv(**x)
    want, last, size = oracle.conv(**x)
    near("y", y, want, size * 1.1, dtype, CONV_UNIT)
    assert torch.equal(final.cpu().double(), last)
    dy, dfinal = m(*y.shape), m(*final.shape)
    got = trunk.conv_backward(dy, **x, dfinal=dfinal)
    grads, sizes = oracle.conv_backward(dy, **x, dfinal=dfinal)
    for name in trunk.ConvGrads._fields:
        near(name, getattr(got, name), grads[name], sizes[name], torch.float32 if name in ("dweight", "dbias") else dtype,
             CONV_UNIT + (199 * 2.0 ** -24 if name in ("dweight", "dbias") else 0))


# ---------------------------------------------------------------------------------------------
# Graphs.


def test_a_graph_replays_every_operator(dtype):
    """Forward, backward and steps captured once, replayed with new inputs and eager work between."""
    x, m = scan_case(dtype, [600, 64, 40], 2, 1, 32, 32, initial=True)
    c, _ = conv_case(dtype, [600, 64, 40], 64, 4, True)
    dy, dyc = m(*x["x"].shape), m(704, 64)
    post, pre = m.f32(64), m.f32(64)
    states, held = m.f32(8, 2, 32, 32), m(8, 3, 64)

    def work(states, held):
        one = {k: x[k][:5] for k in ("x", "dt", "B", "C")}
        return (*trunk.scan(**x), *trunk.scan_backward(dy, **x), *trunk.conv(**c), *trunk.conv_backward(dyc, **c),
                *trunk.norms(c["x"], dyc, post=post, pre=pre), *(g for g in trunk.norms_backward(dyc, c["x"], c["x"], dyc, post=post, pre=pre) if g is not None),
                trunk.scan_step(**one, A=x["A"], states=states), trunk.conv_step(c["x"][:5], c["weight"], held))

    work(states.clone(), held.clone())
    torch.cuda.synchronize()
    a, b = states.clone(), held.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(a, b)
    for _ in range(3):
        x["x"].copy_(m(*x["x"].shape))
        c["x"].copy_(m(*c["x"].shape))
        a.copy_(states), b.copy_(held)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        s, h = states.clone(), held.clone()
        for one, two in zip(got, work(s, h)):
            assert torch.equal(one, two)
        assert torch.equal(a, s) and torch.equal(b, h)
