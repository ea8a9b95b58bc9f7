"""The float trunk's operators on the GPU (include/uor_trunk.h): the selective state space scan and
its short causal convolution (packed sequences, their gradients, single tokens over device slots),
the norms before and after a block fused with its gate and residual scale (and their gradients), and the
trunk's ends over its vocabulary: the embedding's lookup and gradient, the head's cross entropy with its
gradients and its greedy choice, without keeping the logits.

Every function takes and returns torch tensors on one HIP device, runs on torch's current stream and
waits for nothing. Activations are bfloat16 or float32; parameters, the scan's states and the
parameters' gradients are float32. The embedding's table and the head's matrix are of either type, and
their gradients of theirs. Rows are packed: ``offsets`` (int32, one more than there are
sequences, ascending, on the device) says where each sequence's rows begin; without it all rows are
one sequence. Rows before the first offset and from the last one on are no sequence's: what is
returned is 0 there, and nothing else depends on them. Where the inner axes of a tensor are not dense
it is copied first. Errors raise ``TrunkError``; there is no fallback: a missing library or device
raises.

``scan``, ``conv``, ``norms``, ``embed`` and ``loss`` take part in autograd: where an input requires a gradient, the outputs
have ``*_backward`` as theirs, which computes the gradients from the call's own inputs, and which a
program may call by itself (it is not differentiable). The steps update their states in place and have
no gradient, nor has ``choose``: going back through one raises, and so does a forward-mode derivative of
any call. Nothing is kept between calls. Results are the same each time, bit for bit.

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
           "uor_trunk_norms_backward_async", "uor_trunk_sizeof_embed", "uor_trunk_sizeof_head", "uor_trunk_embed_async",
           "uor_trunk_embed_backward_workspace_bytes", "uor_trunk_embed_backward_async", "uor_trunk_loss_workspace_bytes",
           "uor_trunk_loss_async", "uor_trunk_loss_backward_workspace_bytes", "uor_trunk_loss_backward_async",
           "uor_trunk_choose_workspace_bytes", "uor_trunk_choose_async")
ABI_VERSION = 1
DTYPES = {torch.bfloat16: 0, torch.float32: 1}
MAX_DIM = MAX_STATE = 128
MAX_TAPS = 4
MAX_WIDTH = 8192
MAX_VOCAB, MAX_ROWS = 1 << 23, 1 << 24

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


class CEmbed(C.Structure):
    _fields_ = ([("device", C.c_int32)] + [(n, U32) for n in ("dtype", "table_dtype", "rows", "vocab", "width", "wide")] + [("scale", F32)]
                + [(n, I64) for n in ("table_stride", "dy_stride")] + [(n, P) for n in ("tokens", "table", "y", "dy", "dtable")])


class CHead(C.Structure):
    _fields_ = ([("device", C.c_int32)] + [(n, U32) for n in ("dtype", "dweight_dtype", "rows", "vocab", "width", "wide", "reserved")]
                + [(n, I64) for n in ("x_stride", "w_stride")]
                + [(n, P) for n in ("x", "weight", "targets", "losses", "lse", "tokens", "logprobs", "dlosses", "dlse", "dx", "dweight")])


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


class LossGrads(NamedTuple):
    dx: Optional[torch.Tensor]
    dweight: Optional[torch.Tensor]


_Tensor = torch.Tensor
_forward = torch.autograd.forward_ad
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # none without a HIP device to call it for
# Arguments and, of each call that takes them, whether it wants scratch memory.
_FORMS = (("scan", CScan, {"scan": True, "scan_backward": True, "scan_step": False}),
          ("conv", CConv, {"conv": False, "conv_backward": True, "conv_step": False}),
          ("norms", CNorms, {"norms": False, "norms_backward": True}),
          ("embed", CEmbed, {"embed": False, "embed_backward": True}),
          ("head", CHead, {"loss": True, "loss_backward": True, "choose": True}))
_lib = None
_calls = {}  # name: (the call, its workspace's size or None)


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise TrunkError(f"{LIB_PATH} is not built (make -C uor-r4_amd/csrc)")
        L = C.CDLL(LIB_PATH)
        try:
            _bind(L)
        except AttributeError:  # a call that it does not have
            raise TrunkError(f"{LIB_PATH} is of another version: build it again") from None
        _lib = L
    return _lib


def _bind(L):
    """The library's calls and what they take."""
    L.uor_trunk_abi_version.restype = U32
    L.uor_trunk_last_error.restype = C.c_char_p
    for name, struct, forms in _FORMS:
        size = getattr(L, f"uor_trunk_sizeof_{name}")
        size.restype = C.c_uint64
        if size() != C.sizeof(struct) or L.uor_trunk_abi_version() != ABI_VERSION:
            raise TrunkError(f"{LIB_PATH} is of another version: build it again")
        for form, needs in forms.items():
            call, bytes_of = getattr(L, f"uor_trunk_{form}_async"), None
            call.argtypes = [C.POINTER(struct)] + ([P, C.c_uint64] if needs else []) + [P]
            if needs:
                bytes_of = getattr(L, f"uor_trunk_{form}_workspace_bytes")
                bytes_of.argtypes, bytes_of.restype = [C.POINTER(struct)], C.c_uint64
            _calls[form] = call, bytes_of


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


def _no_tangents(tensors):
    """No call has a forward-mode derivative: one that is asked for would be lost."""
    if _forward._current_level >= 0:
        for t in tensors:
            _want(t is None or _forward.unpack_dual(t).tangent is None, "forward-mode derivatives are not computed")


def _one_device(*tensors):
    """The index of the tensors' device: one HIP device for all of them."""
    _no_tangents(tensors)
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
                _no_tangents(tensors)
                return True
    return False


_IN_PLACE = "its states are updated in place"


class _NoGradient(torch.autograd.Function):
    """The outputs of a call that has no gradient, and why."""

    @staticmethod
    def forward(ctx, name, why, call, *inputs):
        ctx.text = f"{name} has no gradient: {why}"
        return call()

    @staticmethod
    def backward(ctx, *grads):
        raise TrunkError(ctx.text)


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
        return _NoGradient.apply("scan_step", _IN_PLACE, lambda: scan_step(x, dt, A, B, C, states, slots=slots, D=D, dt_bias=dt_bias), states, *keep)
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
        return _NoGradient.apply("conv_step", _IN_PLACE, lambda: conv_step(x, weight, states, bias, slots=slots, silu=silu), states, *keep)
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


# ---------------------------------------------------------------------------------------------
# The ends: the embedding, and the head's loss and choice.


def _places(name, t, rows=None):
    """A dense vector of tokens or targets, int32 or int64, and whether it is int64."""
    _want(isinstance(t, _Tensor), "{} is no tensor", name)
    _want(t.dtype in (torch.int32, torch.int64), "{} is {}, not int32 or int64", name, t.dtype)
    _want(t.dim() == 1 if rows is None else t.shape == (rows,), "{} has shape {}, not {}", name, tuple(t.shape), ("rows",) if rows is None else (rows,))
    return (t if t.is_contiguous() else t.contiguous()), int(t.dtype == torch.int64)


def _matrix(name, t):
    """The type, vocabulary and width of a table or a head's matrix."""
    dtype = _dtype(t, name)
    _want(t.dim() == 2, "{} has the axes word and value", name)
    vocab, width = t.shape
    _want(1 <= vocab <= MAX_VOCAB and 1 <= width <= MAX_WIDTH, "{} of {} words of {} values: at most {} of {}, and one of each", name, vocab, width,
          MAX_VOCAB, MAX_WIDTH)
    return dtype, vocab, width


def _embed_args(tokens, table, scale, dtype):
    kind, vocab, width = _matrix("table", table)
    dtype = kind if dtype is None else dtype
    _want(dtype in DTYPES, "dtype is {}, not bfloat16 or float32", dtype)
    tokens, wide = _places("tokens", tokens)
    rows = tokens.numel()
    _want(rows <= MAX_ROWS, "{} rows are more than {}", rows, MAX_ROWS)
    return CEmbed(0, DTYPES[dtype], DTYPES[kind], rows, vocab, width, wide, scale, 0, 0, _ptr(tokens)), tokens, dtype


def embed(tokens, table, *, scale=1.0, dtype=None):
    """y (rows, width) = scale table[tokens], rounded once to ``dtype`` (None: the table's). ``table``
    (vocab, width) is float32 or bfloat16, ``tokens`` (rows) int32 or int64. A token outside the
    vocabulary (padding) has a row of zeros and no part in the gradient."""
    a, tokens, dtype = _embed_args(tokens, table, scale, dtype)
    if _tracked((table,)):
        return _Embed.apply(tokens, table, scale, dtype)
    table, a.table_stride = _rows("table", table, table.dtype, table.shape, a.width)
    index = _one_device(tokens, table)
    y = torch.empty((a.rows, a.width), dtype=dtype, device=table.device)
    a.table, a.y = _ptr(table), _ptr(y)
    _call("embed", a, index)
    return y


def embed_backward(dy, tokens, table, *, scale=1.0):
    """The gradient of ``embed`` at its table, of the table's shape and type: scale times the sums of dy's
    rows by their token, in 32 bits and the rows' order, rounded once. Nothing of ``table`` is read."""
    _want(dy is not None, "dy is no tensor")
    a, tokens, dtype = _embed_args(tokens, table, scale, _dtype(dy, "dy"))
    dy, a.dy_stride = _rows("dy", dy, dtype, (a.rows, a.width), a.width)
    index = _one_device(dy, tokens, table)
    got = _make(table)
    a.dy, a.dtable = _ptr(dy), _ptr(got)
    _call("embed_backward", a, index)
    return got


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale, dtype):
        ctx.save_for_backward(tokens)
        ctx.scale, ctx.table = scale, (table.shape, table.dtype, table.device)  # the table itself may change before the gradient
        return embed(tokens, table, scale=scale, dtype=dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        tokens, = ctx.saved_tensors
        shape, dtype, device = ctx.table
        like = torch.empty((), dtype=dtype, device=device).expand(shape)
        return None, embed_backward(dy, tokens, like, scale=ctx.scale), None, None


def _head_args(x, weight, targets):
    dtype, vocab, width = _matrix("weight", weight)
    _want(isinstance(x, _Tensor) and x.dim() == 2, "x has the axes row and value")
    rows = x.shape[0]
    _want(rows <= MAX_ROWS, "{} rows are more than {}", rows, MAX_ROWS)
    x, xs = _rows("x", x, dtype, (rows, width), width)
    weight, ws = _rows("weight", weight, dtype, (vocab, width), width)
    targets, wide = (None, 0) if targets is None else _places("targets", targets, rows)
    return CHead(0, DTYPES[dtype], DTYPES[dtype], rows, vocab, width, wide, 0, xs, ws, _ptr(x), _ptr(weight), _ptr(targets)), (x, weight, targets)


def loss(x, weight, targets):
    """(losses, lse), float32 (rows): the softmax cross entropy of each row of x (rows, width) over the words of
    ``weight`` (vocab, width; x's type), and the logarithm of its sum, without keeping the logits. ``targets``
    (rows; int32 or int64) says each row's word; a row whose target is outside the vocabulary takes no part, and
    both are 0 there. What is wanted of the losses (their mean over the rows with a target) is the caller's."""
    _want(targets is not None, "targets is no tensor")
    a, keep = _head_args(x, weight, targets)
    if _tracked((x, weight)):
        return _Loss.apply(x, weight, targets)
    index = _one_device(*keep)
    losses, lse = (torch.empty(a.rows, dtype=torch.float32, device=x.device) for _ in range(2))
    a.losses, a.lse = _ptr(losses), _ptr(lse)
    _call("loss", a, index)
    return losses, lse


def loss_backward(dlosses, x, weight, targets, lse, *, dlse=None, dtype=None, dx=True, dweight=True):
    """(dx, dweight): the gradients of ``loss`` at x and weight from those of its outputs (either may be None
    for zeros) and the call's own ``lse``; with ``dx`` or ``dweight`` false that one is None and not computed. The
    logits are computed again, a piece of the vocabulary and of the rows at a time; their gradient, but for the
    targets', is rounded to x's type before its products with x and weight, which are summed in 32 bits.
    ``dtype``: dweight's type, weight's own without (float32 for a program that adds up
    gradients of bfloat16 calls)."""
    _want(targets is not None, "targets is no tensor")
    a, keep = _head_args(x, weight, targets)
    _want(lse is not None, "lse is no tensor")
    lse, dlosses, dlse = (_dense(n, t, torch.float32, (a.rows,)) for n, t in (("lse", lse), ("dlosses", dlosses), ("dlse", dlse)))
    dtype = weight.dtype if dtype is None else dtype
    _want(dtype in DTYPES, "dtype is {}, not bfloat16 or float32", dtype)
    index = _one_device(lse, dlosses, dlse, *keep)
    got = LossGrads(_make(x) if dx else None, torch.empty(weight.shape, dtype=dtype, device=weight.device) if dweight else None)
    a.lse, a.dlosses, a.dlse, a.dweight_dtype = _ptr(lse), _ptr(dlosses), _ptr(dlse), DTYPES[dtype]
    a.dx, a.dweight = map(_ptr, got)
    _call("loss_backward", a, index)
    return got


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets):
        losses, lse = loss(x, weight, targets)
        ctx.save_for_backward(x, weight, targets, lse)
        ctx.set_materialize_grads(False)
        return losses, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlosses, dlse):
        if dlosses is None and dlse is None:
            return None, None, None
        x, weight, targets, lse = ctx.saved_tensors
        dx, dweight, _ = ctx.needs_input_grad
        got = loss_backward(dlosses, x, weight, targets, lse, dlse=dlse, dx=dx, dweight=dweight)
        return got.dx, got.dweight, None


def choose(x, weight):
    """(tokens, logprobs): of each row of x (rows, width) the word of ``weight`` (vocab, width; x's type) with the
    largest logit, the lowest of equals (int64), and its log probability (float32), without keeping the logits. The
    log probability has no gradient: going back through it raises (``loss`` of the tokens has one). Of a row with no
    logit over -inf the token is 0; logits that are no number are not chosen."""
    a, keep = _head_args(x, weight, None)
    if _tracked((x, weight)):
        return _NoGradient.apply("choose", "loss gives a token's log probability with one", lambda: choose(x, weight), x, weight)
    index = _one_device(*keep)
    tokens = torch.empty(a.rows, dtype=torch.int64, device=x.device)
    logprobs = torch.empty(a.rows, dtype=torch.float32, device=x.device)
    a.tokens, a.logprobs = _ptr(tokens), _ptr(logprobs)
    _call("choose", a, index)
    return tokens, logprobs
