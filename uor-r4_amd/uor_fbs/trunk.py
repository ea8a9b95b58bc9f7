"""The float trunk's operators on the GPU (include/uor_trunk.h): the selective state space scan and
its short causal convolution (packed sequences, their gradients, single tokens over device slots),
and the norms before and after a block fused with its gate and residual scale (and their gradients).

Every function takes and returns torch tensors on one HIP device, runs on torch's current stream and
waits for nothing. Activations are bfloat16 or float32; parameters, the scan's states and the
parameters' gradients are float32. Rows are packed: ``offsets`` (int32, one more than there are
sequences, ascending, on the device) says where each sequence's rows begin; without it all rows are
one sequence. Rows before the first offset and from the last one on are no sequence's: what is
returned is 0 there, and nothing else depends on them. Where the inner axes of a tensor are not dense
it is copied first. Errors raise ``TrunkError``; there is no fallback: a missing library or device
raises.

``scan``, ``conv`` and ``norms`` take part in autograd: where an input requires a gradient, the outputs
have ``*_backward`` as theirs, which computes the gradients from the call's own inputs, and which a
program may call by itself (it is not differentiable). The steps update their states in place and have
no gradient: going back through one raises. Nothing is kept between calls. Results are the same each
time, bit for bit.

A training step that is captured into a graph calls ``*_backward`` by itself, or has no eager graph of the
same leaves alive meanwhile: torch would order their gradients after the other graph's stream.
"""

from __future__ import annotations

import ctypes as C
import os
from typing import NamedTuple, Optional

import torch

PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(PKG, "lib", "libuor_trunk_hip.so")
SYMBOLS = ("uor_trunk_abi_version", "uor_trunk_last_error", "uor_trunk_sizeof_scan", "uor_trunk_sizeof_conv",
           "uor_trunk_sizeof_norms", "uor_trunk_scan_workspace_bytes", "uor_trunk_scan_async",
           "uor_trunk_scan_backward_workspace_bytes", "uor_trunk_scan_backward_async", "uor_trunk_scan_step_async",
           "uor_trunk_conv_async", "uor_trunk_conv_backward_workspace_bytes", "uor_trunk_conv_backward_async",
           "uor_trunk_conv_step_async", "uor_trunk_norms_async", "uor_trunk_norms_backward_workspace_bytes",
           "uor_trunk_norms_backward_async")
ABI_VERSION = 1
DTYPES = {torch.bfloat16: 0, torch.float32: 1}
MAX_DIM = MAX_STATE = 128
MAX_TAPS = 4
MAX_WIDTH = 8192

P, I64, U32, F32 = C.c_void_p, C.c_int64, C.c_uint32, C.c_float


class TrunkError(ValueError):
    pass


class CScan(C.Structure):
    _fields_ = ([("device", C.c_int32)] + [(n, U32) for n in ("dtype", "tokens", "seqs", "heads", "groups", "dim", "state",
                                                              "slots", "reserved")]
                + [(n, I64) for n in ("x_stride", "dt_stride", "b_stride", "c_stride", "y_stride")]
                + [(n, P) for n in ("x", "dt", "B", "C", "A", "D", "dt_bias", "offsets", "initial", "y", "final", "index",
                                    "states", "dy", "dfinal", "dx", "ddt", "dB", "dC", "dA", "dD", "ddt_bias", "dinitial")])


class CConv(C.Structure):
    _fields_ = ([("device", C.c_int32)] + [(n, U32) for n in ("dtype", "tokens", "seqs", "channels", "taps", "slots", "silu")]
                + [(n, I64) for n in ("x_stride", "y_stride")]
                + [(n, P) for n in ("x", "weight", "bias", "offsets", "initial", "y", "final", "index", "states", "dy",
                                    "dfinal", "dx", "dinitial", "dweight", "dbias")])


class CNorms(C.Structure):
    _fields_ = ([("device", C.c_int32)] + [(n, U32) for n in ("dtype", "rows", "width")] + [("eps", F32), ("reserved", U32)]
                + [(n, I64) for n in ("residual_stride", "out_stride", "gate_stride")]
                + [(n, P) for n in ("residual", "out", "gate", "post", "scale", "pre", "residual_out", "normed",
                                    "dresidual_out", "dnormed", "dresidual", "dout", "dgate", "dpost", "dscale", "dpre")])


class ScanGrads(NamedTuple):
    dx: torch.Tensor
    ddt: torch.Tensor
    dA: torch.Tensor
    dB: torch.Tensor
    dC: torch.Tensor
    dD: Optional[torch.Tensor]
    ddt_bias: Optional[torch.Tensor]
    dinitial: Optional[torch.Tensor]


class ConvGrads(NamedTuple):
    dx: torch.Tensor
    dweight: torch.Tensor
    dbias: Optional[torch.Tensor]
    dinitial: Optional[torch.Tensor]


class NormGrads(NamedTuple):
    dresidual: Optional[torch.Tensor]
    dout: Optional[torch.Tensor]
    dgate: Optional[torch.Tensor]
    dpost: Optional[torch.Tensor]
    dscale: Optional[torch.Tensor]
    dpre: Optional[torch.Tensor]


_Tensor = torch.Tensor
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # none without a HIP device to call it for
_lib = None
_calls = {}  # name: (the call, its workspace's size or None)


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise TrunkError(f"{LIB_PATH} is not built (make -C uor-r4_amd/csrc)")
        L = C.CDLL(LIB_PATH)
        L.uor_trunk_abi_version.restype = U32
        L.uor_trunk_last_error.restype = C.c_char_p
        for name, struct in (("scan", CScan), ("conv", CConv), ("norms", CNorms)):
            size = getattr(L, f"uor_trunk_sizeof_{name}")
            size.restype = C.c_uint64
            if size() != C.sizeof(struct) or L.uor_trunk_abi_version() != ABI_VERSION:
                raise TrunkError(f"{LIB_PATH} is of another version: build it again")
            forms = {"scan": ("", "_backward", "_step"), "conv": ("", "_backward", "_step"), "norms": ("", "_backward")}[name]
            for form in forms:
                call, bytes_of = getattr(L, f"uor_trunk_{name}{form}_async"), None
                needs = form == "_backward" or (name == "scan" and form == "")
                call.argtypes = [C.POINTER(struct)] + ([P, C.c_uint64] if needs else []) + [P]
                if needs:
                    bytes_of = getattr(L, f"uor_trunk_{name}{form}_workspace_bytes")
                    bytes_of.argtypes, bytes_of.restype = [C.POINTER(struct)], C.c_uint64
                _calls[name + form] = call, bytes_of
        _lib = L
    return _lib


def _call(name, args, index):
    """The library's call on the current stream of device `index`."""
    L = _lib or lib()
    call, bytes_of = _calls[name]
    args.device, ref, stream = index, C.byref(args), _raw_stream(index)
    if bytes_of is None:
        code = call(ref, stream)
    else:
        n = bytes_of(ref)
        keep = torch.empty(n, dtype=torch.uint8, device=torch.device("cuda", index)) if n else None
        code = call(ref, None if keep is None else keep.data_ptr(), n, stream)
    if code:
        raise TrunkError(f"uor_trunk_{name} status {code}: {L.uor_trunk_last_error().decode()}")


def _want(ok, text, *values):
    if not ok:
        raise TrunkError(text.format(*values))


def _check(name, t, dtype, shape):
    _want(isinstance(t, torch.Tensor), "{} is no tensor", name)
    _want(t.dtype == dtype, "{} is {}, not {}", name, t.dtype, dtype)
    _want(t.shape == shape, "{} has shape {}, not {}", name, tuple(t.shape), shape)


def _rows(name, t, dtype, shape, inner):
    """t with dense inner axes of `inner` values, and the values between its rows (None: None, 0)."""
    if t is None:
        return None, 0
    if not (isinstance(t, _Tensor) and t.dtype is dtype and t.shape == shape):
        _check(name, t, dtype, shape)
    if t.is_contiguous():
        return t, inner
    size_so_far = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != size_so_far:
            return t.contiguous(), inner
        size_so_far *= size
    if t.shape[0] > 1 and t.stride(0) < inner:
        return t.contiguous(), inner
    return t, (t.stride(0) if t.shape[0] > 1 else inner)


def _dense(name, t, dtype, shape):
    if t is None:
        return None
    if not (isinstance(t, _Tensor) and t.dtype is dtype and t.shape == shape):
        _check(name, t, dtype, shape)
    return t if t.is_contiguous() else t.contiguous()


def _one_device(*tensors):
    """The index of the tensors' device: one HIP device for all of them."""
    index = None
    for t in tensors:
        if t is not None:
            at = t.get_device()
            if index is None:
                index = at
            elif at != index:
                raise TrunkError("the tensors are on different devices: {}".format(sorted({str(t.device) for t in tensors if t is not None})))
    _want(index is not None and index >= 0, "the tensors are on cpu: a HIP device is wanted")
    return index


def _offsets(offsets, tokens):
    if offsets is None:
        return None, 1
    _want(isinstance(offsets, torch.Tensor), "offsets is no tensor")
    _want(offsets.dim() == 1 and offsets.numel() >= 2, "offsets has one place more than there are sequences, two at least")
    return _int32("offsets", offsets), offsets.numel() - 1


def _int32(name, t):
    _want(t.dtype in (torch.int32, torch.int64), "{} is {}, not int32", name, t.dtype)
    t = t if t.dtype == torch.int32 else t.clamp(-1, 2 ** 31 - 1).int()  # what is outside stays outside
    return t if t.is_contiguous() else t.contiguous()


def _index(slots, rows, states):
    if slots is None:
        _want(states >= rows, "{} rows for {} states", rows, states)
        return None
    _want(isinstance(slots, torch.Tensor), "slots is no tensor")
    _want(slots.shape == (rows,), "slots has shape {}, not {}", tuple(slots.shape), (rows,))
    return _int32("slots", slots)


_NOTHING = 16  # the address of a tensor of no values: it is there, and nothing of it is read


def _ptr(t):
    return None if t is None else t.data_ptr() or _NOTHING


def _dtype(t, name):
    _want(isinstance(t, torch.Tensor) and t.dtype in DTYPES, "{} is no tensor of bfloat16 or float32", name)
    return t.dtype


def _make(like):
    """A dense tensor of the same type, shape and device (None: None)."""
    if like is None:
        return None
    return torch.empty_like(like) if like.is_contiguous() else torch.empty_like(like, memory_format=torch.contiguous_format)


def _tracked(tensors):
    """Whether a gradient is wanted at one of them."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


class _Step(torch.autograd.Function):
    """A step's outputs, of which there is no gradient."""

    @staticmethod
    def forward(ctx, name, call, *inputs):
        ctx.name = name
        return call()

    @staticmethod
    def backward(ctx, *grads):
        raise TrunkError(f"{ctx.name} has no gradient: its states are updated in place")


_changed = torch.autograd.graph.increment_version  # of states in place, for autograd to see


# ---------------------------------------------------------------------------------------------
# The scan.


def _scan_args(x, dt, A, B, Cm, D, dt_bias, offsets, initial, step=False):
    dtype = _dtype(x, "x")
    _want(x.dim() == 3, "x has the axes row, head and value")
    _want(isinstance(B, torch.Tensor) and B.dim() == 3, "B has the axes row, group and state")
    tokens, heads, dim = x.shape
    _, groups, state = B.shape
    _want(groups >= 1 and heads >= 1 and heads % groups == 0, "{} heads are not whole groups of {}", heads, groups)
    _want(1 <= dim <= MAX_DIM and 1 <= state <= MAX_STATE, "dim {} or state {} outside 1..128", dim, state)
    off, seqs = (None, tokens) if step else _offsets(offsets, tokens)
    x, xs = _rows("x", x, dtype, (tokens, heads, dim), heads * dim)
    dt, ds = _rows("dt", dt, dtype, (tokens, heads), heads)
    B, bs = _rows("B", B, dtype, (tokens, groups, state), groups * state)
    Cm, cs = _rows("C", Cm, dtype, (tokens, groups, state), groups * state)
    f32 = torch.float32
    _want(A is not None, "A is no tensor")
    A, D, dt_bias = _dense("A", A, f32, (heads,)), _dense("D", D, f32, (heads,)), _dense("dt_bias", dt_bias, f32, (heads,))
    initial = _dense("initial", initial, f32, (seqs, heads, dim, state))
    a = CScan(0, DTYPES[dtype], tokens, seqs, heads, groups, dim, state, 0, 0, xs, ds, bs, cs, heads * dim, _ptr(x), _ptr(dt),
              _ptr(B), _ptr(Cm), _ptr(A), _ptr(D), _ptr(dt_bias), _ptr(off), _ptr(initial))
    return a, (x, dt, A, B, Cm, D, dt_bias, off, initial)


def scan(x, dt, A, B, C, *, D=None, dt_bias=None, offsets=None, initial=None):
    """(y, final): the scan of x (rows, heads, dim) with dt (rows, heads), A (heads), B and C (rows,
    groups, state), the skip D and the steps' bias (heads), from the states ``initial`` (sequences,
    heads, dim, state; zeros without). ``final`` are the states after each sequence's last row."""
    a, keep = _scan_args(x, dt, A, B, C, D, dt_bias, offsets, initial)
    if _tracked(keep):
        return _Scan.apply(x, dt, A, B, C, D, dt_bias, offsets, initial)
    index = _one_device(*keep)
    y, final = _make(x), torch.empty((a.seqs, a.heads, a.dim, a.state), dtype=torch.float32, device=x.device)
    a.y, a.final = _ptr(y), _ptr(final)
    _call("scan", a, index)
    return y, final


def scan_backward(dy, x, dt, A, B, C, *, D=None, dt_bias=None, offsets=None, initial=None, dfinal=None):
    """The gradients of ``scan`` at its inputs from those of its outputs; ``dfinal`` None: zeros.
    dD, ddt_bias and dinitial are None where the input is."""
    a, keep = _scan_args(x, dt, A, B, C, D, dt_bias, offsets, initial)
    _want(dy is not None, "dy is no tensor")
    dy, a.y_stride = _rows("dy", dy, x.dtype, x.shape, a.heads * a.dim)
    dfinal = _dense("dfinal", dfinal, torch.float32, (a.seqs, a.heads, a.dim, a.state))
    index = _one_device(dy, dfinal, *keep)
    got = ScanGrads(*map(_make, (x, dt, A, B, C, D, dt_bias, initial)))
    a.dy, a.dfinal = _ptr(dy), _ptr(dfinal)
    a.dx, a.ddt, a.dA, a.dB, a.dC, a.dD, a.ddt_bias, a.dinitial = map(_ptr, got)
    _call("scan_backward", a, index)
    return got


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, dt_bias, offsets, initial):
        ctx.save_for_backward(x, dt, A, B, C, D, dt_bias, offsets, initial)
        ctx.set_materialize_grads(False)
        return scan(x, dt, A, B, C, D=D, dt_bias=dt_bias, offsets=offsets, initial=initial)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfinal):
        if dy is None and dfinal is None:
            return (None,) * 9
        x, dt, A, B, C, D, dt_bias, offsets, initial = ctx.saved_tensors
        got = scan_backward(torch.zeros_like(x) if dy is None else dy, x, dt, A, B, C, D=D, dt_bias=dt_bias, offsets=offsets,
                            initial=initial, dfinal=dfinal)
        return got.dx, got.ddt, got.dA, got.dB, got.dC, got.dD, got.ddt_bias, None, got.dinitial


def scan_step(x, dt, A, B, C, states, *, slots=None, D=None, dt_bias=None):
    """y (rows, heads, dim): one token a session. ``states`` (slots, heads, dim, state) float32 is
    updated in place; ``slots`` (int32) says which state each row has, no two alike. A row whose slot
    is outside the states is skipped and its y is 0."""
    a, keep = _scan_args(x, dt, A, B, C, D, dt_bias, None, None, step=True)
    inner = (a.heads, a.dim, a.state)
    _want(isinstance(states, torch.Tensor) and states.dtype == torch.float32 and states.dim() == 4 and states.shape[1:] == inner
          and states.is_contiguous(), "states is no dense float32 tensor of (slots, {}, {}, {})", *inner)
    if _tracked((states, *keep)):
        return _Step.apply("scan_step", lambda: scan_step(x, dt, A, B, C, states, slots=slots, D=D, dt_bias=dt_bias), states, *keep)
    slots = _index(slots, a.tokens, states.shape[0])
    index = _one_device(states, slots, *keep)
    y = _make(x)
    a.y, a.index, a.states, a.slots = _ptr(y), _ptr(slots), _ptr(states), states.shape[0]
    _call("scan_step", a, index)
    _changed((states,))
    return y


# ---------------------------------------------------------------------------------------------
# The convolution.


def _conv_args(x, weight, bias, offsets, initial, silu, step=False):
    dtype = _dtype(x, "x")
    _want(x.dim() == 2, "x has the axes row and channel")
    _want(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight has the axes channel and tap")
    tokens, channels = x.shape
    taps = weight.shape[1]
    _want(channels >= 1 and 1 <= taps <= MAX_TAPS, "{} taps outside 1..{}, or no channels", taps, MAX_TAPS)
    off, seqs = (None, tokens) if step else _offsets(offsets, tokens)
    x, xs = _rows("x", x, dtype, (tokens, channels), channels)
    weight = _dense("weight", weight, torch.float32, (channels, taps))
    bias = _dense("bias", bias, torch.float32, (channels,))
    initial = _dense("initial", initial, dtype, (seqs, taps - 1, channels))
    a = CConv(0, DTYPES[dtype], tokens, seqs, channels, taps, 0, 1 if silu else 0, xs, channels, _ptr(x), _ptr(weight), _ptr(bias),
              _ptr(off), _ptr(initial))
    return a, (x, weight, bias, off, initial)


def conv(x, weight, bias=None, *, offsets=None, initial=None, silu=True):
    """(y, final): y_t = silu(bias + sum_k weight[:, k] x_(t - taps + 1 + k)) over each sequence's own
    rows of x (rows, channels), the rows before it from ``initial`` (sequences, taps - 1, channels;
    zeros without). ``final`` are each sequence's last taps - 1 rows, the next call's ``initial``."""
    a, keep = _conv_args(x, weight, bias, offsets, initial, silu)
    if _tracked(keep):
        return _Conv.apply(x, weight, bias, offsets, initial, silu)
    index = _one_device(*keep)
    y, final = _make(x), torch.empty((a.seqs, a.taps - 1, a.channels), dtype=x.dtype, device=x.device)
    a.y, a.final = _ptr(y), _ptr(final)
    _call("conv", a, index)
    return y, final


def conv_backward(dy, x, weight, bias=None, *, offsets=None, initial=None, dfinal=None, silu=True):
    """The gradients of ``conv`` at its inputs; dbias and dinitial are None where the input is."""
    a, keep = _conv_args(x, weight, bias, offsets, initial, silu)
    _want(dy is not None, "dy is no tensor")
    dy, a.y_stride = _rows("dy", dy, x.dtype, x.shape, a.channels)
    dfinal = _dense("dfinal", dfinal, x.dtype, (a.seqs, a.taps - 1, a.channels))
    index = _one_device(dy, dfinal, *keep)
    got = ConvGrads(*map(_make, (x, weight, bias, initial)))
    a.dy, a.dfinal = _ptr(dy), _ptr(dfinal)
    a.dx, a.dweight, a.dbias, a.dinitial = map(_ptr, got)
    _call("conv_backward", a, index)
    return got


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets, initial, silu):
        ctx.save_for_backward(x, weight, bias, offsets, initial)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return conv(x, weight, bias, offsets=offsets, initial=initial, silu=silu)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfinal):
        if dy is None and dfinal is None:
            return (None,) * 6
        x, weight, bias, offsets, initial = ctx.saved_tensors
        got = conv_backward(torch.zeros_like(x) if dy is None else dy, x, weight, bias, offsets=offsets, initial=initial, dfinal=dfinal,
                            silu=ctx.silu)
        return got.dx, got.dweight, got.dbias, None, got.dinitial, None


def conv_step(x, weight, states, bias=None, *, slots=None, silu=True):
    """y (rows, channels): one token a session; ``states`` (slots, taps - 1, channels) of x's type is
    updated in place, ``slots`` as in ``scan_step``."""
    a, keep = _conv_args(x, weight, bias, None, None, silu, step=True)
    inner = (a.taps - 1, a.channels)
    _want(isinstance(states, torch.Tensor) and states.dtype == x.dtype and states.dim() == 3 and states.shape[1:] == inner
          and states.is_contiguous(), "states is no dense {} tensor of (slots, {}, {})", x.dtype, *inner)
    if _tracked((states, *keep)):
        return _Step.apply("conv_step", lambda: conv_step(x, weight, states, bias, slots=slots, silu=silu), states, *keep)
    slots = _index(slots, a.tokens, states.shape[0])
    index = _one_device(states, slots, *keep)
    y = _make(x)
    a.y, a.index, a.states, a.slots = _ptr(y), _ptr(slots), _ptr(states), states.shape[0]
    _call("conv_step", a, index)
    _changed((states,))
    return y


# ---------------------------------------------------------------------------------------------
# The norms.


def _norms_args(residual, out, gate, post, scale, pre, eps):
    first = residual if residual is not None else out
    dtype = _dtype(first, "residual" if residual is not None else "out")
    _want(first.dim() == 2, "rows have the axes row and value")
    _want(out is not None or (gate is None and post is None and scale is None), "a gate, post or scale without a block's output")
    _want(out is not None or pre is not None, "nothing to compute: neither a block's output nor pre")
    rows, width = shape = first.shape
    _want(1 <= width <= MAX_WIDTH, "width {} outside 1..{}", width, MAX_WIDTH)
    _want(eps >= 0, "eps is negative")
    residual, rs = _rows("residual", residual, dtype, shape, width)
    out, os_ = _rows("out", out, dtype, shape, width)
    gate, gs = _rows("gate", gate, dtype, shape, width)
    post, scale, pre = (_dense(n, t, torch.float32, (width,)) for n, t in (("post", post), ("scale", scale), ("pre", pre)))
    a = CNorms(0, DTYPES[dtype], rows, width, eps, 0, rs, os_, gs, _ptr(residual), _ptr(out), _ptr(gate), _ptr(post), _ptr(scale),
               _ptr(pre))
    return a, first, (residual, out, gate, post, scale, pre)


def norms(residual, out=None, *, gate=None, post=None, scale=None, pre=None, eps=1e-6):
    """(residual', normed) between two blocks: v = out silu(gate), residual' = residual + scale
    rms(v) post, normed = rms(residual') pre, with rows of (rows, width). Without ``out`` the residual
    is only normed (residual' is the residual itself); without ``residual`` residual' is the normed
    block alone; without ``pre`` normed is None. ``gate``, ``post`` and ``scale`` are 1 without."""
    a, first, keep = _norms_args(residual, out, gate, post, scale, pre, eps)
    if _tracked(keep):
        residual_out, normed = _Norms.apply(residual, out, gate, post, scale, pre, eps)
        return (residual if out is None else residual_out), normed
    index = _one_device(*keep)
    residual_out = residual if out is None else _make(first)
    normed = None if pre is None else _make(first)
    a.normed = _ptr(normed)
    a.residual_out = None if out is None else _ptr(residual_out)
    _call("norms", a, index)
    return residual_out, normed


def norms_backward(dresidual_out, dnormed, residual, out=None, *, gate=None, post=None, scale=None, pre=None, eps=1e-6):
    """The gradients of ``norms`` at its inputs, None where there is none; either of the outputs'
    gradients may be None for zeros."""
    a, first, keep = _norms_args(residual, out, gate, post, scale, pre, eps)
    _want(dnormed is None or pre is not None, "dnormed without pre")
    dresidual_out = _dense("dresidual_out", dresidual_out, first.dtype, first.shape)
    dnormed = _dense("dnormed", dnormed, first.dtype, first.shape)
    index = _one_device(dresidual_out, dnormed, *keep)
    got = NormGrads(*map(_make, (residual, out, gate, post, scale, pre)))
    a.dresidual_out, a.dnormed = _ptr(dresidual_out), _ptr(dnormed)
    a.dresidual, a.dout, a.dgate, a.dpost, a.dscale, a.dpre = map(_ptr, got)
    _call("norms_backward", a, index)
    return got


class _Norms(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, out, gate, post, scale, pre, eps):
        ctx.save_for_backward(residual, out, gate, post, scale, pre)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        residual_out, normed = norms(residual, out, gate=gate, post=post, scale=scale, pre=pre, eps=eps)
        return (None if out is None else residual_out), normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dresidual_out, dnormed):
        if dresidual_out is None and dnormed is None:
            return (None,) * 7
        residual, out, gate, post, scale, pre = ctx.saved_tensors
        return (*norms_backward(dresidual_out, dnormed, residual, out, gate=gate, post=post, scale=scale, pre=pre, eps=ctx.eps), None)
