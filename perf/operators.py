"""The operators of a float recurrent trunk, as cases that can be timed and compared.

The integer step of this framework serves trunks whose layers are a norm, a causal window of a few
rows, a recurrence with one decay a lane and a gated block between norms. These are the same parts
in floating point, as a program needs them that trains such a trunk or answers with it before it is
exported: the selective state space scan, its short causal convolution, and the norms before and
after a block fused with its gate and residual scale; each over packed sequences of different
lengths, with its gradient, and (the recurrent two) for single tokens over device slots.

``own = False`` computes them in their plain form from elementary torch operations in 32 bits (64
for the sums of logarithms of decays), rounded once at the end. ``own = True`` calls
``uor_fbs.trunk``.

    scan   h_t = exp(D_t A) h_(t-1) + D_t x_t (x) B_t,  y_t = h_t C_t + S x_t,  D_t = softplus(dt_t + bias)
    conv   y_t = silu(bias + sum_k w_k x_(t-K+1+k)), over the sequence's own rows
    norms  v = u silu(z),  r' = r + s rms(v) g_post,  n = rms(r') g_pre
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "uor-r4_amd"))

own = False

EPS = 1e-6
CHUNK = 64  # rows of a chunk in the plain scan


def listed():
    return [
        # Prompts taken in before generation: 300 of up to 509 tokens, packed, at width 256 (inner
        # width 512 as 8 heads of 64).
        dict(name="scan_w256_300x509", op="scan", dtype="bf16", seqs=300, length=509, ragged=True,
             heads=8, groups=1, dim=64, state=64, initial=False),
        # One long document at width 512: few heads, a long axis, resumed from a state.
        dict(name="scan_w512_1x65536", op="scan", dtype="bf16", seqs=1, length=65536, ragged=False,
             heads=16, groups=2, dim=64, state=128, initial=True),
        # A short check in 32 bits at width 128, heads and state of odd sizes.
        dict(name="scan_w128_f32_5x77", op="scan", dtype="f32", seqs=5, length=77, ragged=True,
             heads=6, groups=3, dim=40, state=20, initial=True),
        # A training step's gradients: 2,048 rows of 128 tokens at width 256.
        dict(name="scan_grad_w256_2048x128", op="scan_grad", dtype="bf16", seqs=2048, length=128,
             ragged=False, heads=8, groups=1, dim=64, state=64, initial=False),
        # The gradients of ragged rows in 32 bits, through initial and final states.
        dict(name="scan_grad_f32_37x301", op="scan_grad", dtype="f32", seqs=37, length=301, ragged=True,
             heads=4, groups=2, dim=64, state=32, initial=True),
        # The serving loop: 1,024 sessions take one token each, their states in device slots.
        dict(name="scan_step_w256_b1024", op="scan_step", dtype="bf16", seqs=1024, slots=1100,
             heads=8, groups=1, dim=64, state=64),
        # A few live sessions: latency.
        dict(name="scan_step_w128_b8", op="scan_step", dtype="bf16", seqs=8, slots=16,
             heads=8, groups=1, dim=32, state=32),
        # The prompts' convolution over the scan's inputs (512 channels and two of 64).
        dict(name="conv_w256_300x509", op="conv", dtype="bf16", seqs=300, length=509, ragged=True,
             channels=640, taps=4, initial=False),
        # Its gradient in a training step.
        dict(name="conv_grad_w256_2048x128", op="conv_grad", dtype="bf16", seqs=2048, length=128,
             ragged=False, channels=640, taps=4, initial=False),
        # The serving loop's convolution for single tokens.
        dict(name="conv_step_w256_b1024", op="conv_step", dtype="bf16", seqs=1024, slots=1100,
             channels=640, taps=4),
        # Between two layers of a prompt: the norm after one block, the next one's before.
        dict(name="norms_w256_152700", op="norms", dtype="bf16", rows=152700, width=256, gate=True,
             post=True, pre=True),
        # The same in a training step, backward, at width 512.
        dict(name="norms_grad_w512_131072", op="norms_grad", dtype="bf16", rows=131072, width=512,
             gate=True, post=True, pre=True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan_grad", "scan_grad", "scan_step", "conv", "conv_grad", "conv_step",
                     "norms", "norms_grad"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op.startswith("norms"):
        rows, width = _log(rng, 1, 60000), _log(rng, 8, 4096)
        rows = max(1, min(rows, (1 << 25) // width))
        part = rng.choice(["both", "both", "post", "pre"])
        return dict(op=op, dtype=dtype, rows=rows, width=width, gate=part != "pre" and rng.random() < 0.7,
                    post=part != "pre", pre=part != "post")
    if op.endswith("_step"):
        n = _log(rng, 1, 1024)
        case = dict(op=op, dtype=dtype, seqs=n, slots=n + rng.randrange(0, 40))
    else:
        seqs = _log(rng, 1, 256)
        case = dict(op=op, dtype=dtype, seqs=seqs, length=_log(rng, 1, min(8192, 32768 // seqs)),
                    ragged=rng.random() < 0.7, initial=rng.random() < 0.5)
    if op.startswith("conv"):
        return dict(case, channels=_log(rng, 8, 1536), taps=rng.choice([2, 3, 4, 4]))
    groups = rng.choice([1, 1, 2, 3])
    return dict(case, heads=groups * rng.choice([1, 2, 4, 5]), groups=groups,
                dim=rng.choice([16, 32, 64, 64, 128, rng.randrange(1, 129)]),
                state=rng.choice([16, 32, 64, 128, rng.randrange(1, 129)]))


# ---------------------------------------------------------------------------------------------
# What a program has in hand.


def _lengths(case):
    """The case's lengths: one of them whole, one of nothing where there are more than three."""
    n, most = case["seqs"], case["length"]
    if not case["ragged"]:
        return np.full(n, most)
    lengths = np.random.default_rng(n * 100003 + most).integers(1, most + 1, n)
    lengths[0] = most
    if n > 3:
        lengths[1] = 0
    return lengths


class _Inputs:
    """Tensors made from a seed, on the GPU."""

    def __init__(self, case, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32

    def normal(self, *shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=self.gen) * scale).to(self.dtype)

    def normal32(self, *shape, scale=1.0, mean=0.0):
        return torch.randn(shape, device="cuda", generator=self.gen) * scale + mean

    def uniform32(self, lo, hi, *shape):
        return torch.rand(shape, device="cuda", generator=self.gen) * (hi - lo) + lo


def _offsets(case, seed):
    lengths = np.random.default_rng(seed).permutation(_lengths(case))
    offsets = np.zeros(len(lengths) + 1, np.int32)
    offsets[1:] = np.cumsum(lengths)
    return torch.from_numpy(offsets).cuda()


def _scan_weights(case, i):
    """A (negative), the skip and the steps' bias: the steps lie between 0.001 and 0.1."""
    h = case["heads"]
    step = torch.exp(i.uniform32(math.log(1e-3), math.log(0.1), h))
    return dict(A=-i.uniform32(1.0, 16.0, h), D=i.normal32(h, scale=0.5, mean=1.0),
                dt_bias=step + torch.log(-torch.expm1(-step)))


def prepare(case, seed):
    i, op = _Inputs(case, seed), case["op"]
    s = dict(case)
    if op.startswith("norms"):
        rows, width = case["rows"], case["width"]
        if case["post"]:
            s["residual"], s["out"] = i.normal(rows, width, scale=2.0), i.normal(rows, width)
            s["post"], s["scale"] = i.normal32(width, scale=0.2, mean=1.0), i.normal32(width, scale=0.1, mean=0.5)
        else:
            s["residual"], s["out"], s["post"], s["scale"] = i.normal(rows, width, scale=2.0), None, None, None
        s["gate"] = i.normal(rows, width) if case["gate"] else None
        s["pre"] = i.normal32(width, scale=0.2, mean=1.0) if case["pre"] else None
        if op == "norms_grad":
            s["d_residual"] = i.normal(rows, width)
            s["d_normed"] = i.normal(rows, width) if case["pre"] else None
        return s
    n = case["seqs"]
    if op.endswith("_step"):
        tokens = n
        order = np.random.default_rng(seed).permutation(case["slots"])[:n]
        s["index"] = torch.from_numpy(order.astype(np.int32)).cuda()
    else:
        s["offsets"] = _offsets(case, seed)
        tokens = int(_lengths(case).sum())
    if op.startswith("conv"):
        c, k = case["channels"], case["taps"]
        s.update(x=i.normal(tokens, c), weight=i.normal32(c, k, scale=0.4), bias=i.normal32(c, scale=0.1))
        if op == "conv_step":
            s["held"] = i.normal(case["slots"], k - 1, c)
        else:
            s["start"] = i.normal(n, k - 1, c) if case["initial"] else None
        if op == "conv_grad":
            s["dy"] = i.normal(tokens, c)
            s["d_final"] = i.normal(n, k - 1, c) if case["initial"] else None
        return s
    h, g, p, m = case["heads"], case["groups"], case["dim"], case["state"]
    s.update(_scan_weights(case, i), x=i.normal(tokens, h, p), dt=i.normal(tokens, h, scale=0.5),
             B=i.normal(tokens, g, m, scale=m ** -0.25), C=i.normal(tokens, g, m, scale=m ** -0.25))
    if op == "scan_step":
        s["held"] = i.normal32(case["slots"], h, p, m, scale=0.5)
    else:
        s["start"] = i.normal32(n, h, p, m, scale=0.5) if case["initial"] else None
    if op == "scan_grad":
        s["dy"] = i.normal(tokens, h, p)
        s["d_final"] = i.normal32(n, h, p, m, scale=0.5) if case["initial"] else None
    return s


# ---------------------------------------------------------------------------------------------
# The plain forms, in 32 bits.


def _rows(offsets, length, chunk):
    """Packed rows as (sequence, row) and back: the packed row of each place, whether it is one of
    the sequence's own, and the place of each packed row."""
    total = -(-length // chunk) * chunk
    at = offsets[:-1, None].long() + torch.arange(total, device="cuda")
    valid = at < offsets[1:, None]
    return at, valid, total


def _places(offsets, tokens, total):
    t = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(offsets[1:].contiguous(), t.int(), right=True)
    return seq * total + t - offsets[seq].long()


def _unpack(x, at, valid):
    """x's rows as (sequence, row, ...), zeros where a sequence has none."""
    rows = x[at.clamp(max=max(x.shape[0] - 1, 0))]
    return rows.masked_fill(~valid.reshape(valid.shape + (1,) * (x.dim() - 1)), 0)


def _scan_plain(x, dt, A, B, C, D, bias, offsets, start, length):
    """The scan by chunks: products within a chunk, and the chunks' states joined by a product
    with their decays. Everything in 32 bits but the sums of the decays' logarithms."""
    tokens, heads, dim = x.shape
    groups, width = B.shape[1:]
    chunk = min(CHUNK, length)
    at, valid, total = _rows(offsets, length, chunk)
    seqs, chunks, share = at.shape[0], total // chunk, heads // groups
    cut = lambda v: _unpack(v, at, valid).reshape(seqs, chunks, chunk, *v.shape[1:])  # noqa: E731
    step = cut(F.softplus(dt + bias))  # (seqs, chunks, chunk, heads)
    xs, bs, cs = cut(x), cut(B), cut(C)
    log = torch.cumsum((step.double() * A.double()), 2).permute(0, 1, 3, 2)  # (seqs, chunks, heads, chunk)
    later = torch.ones(chunk, chunk, dtype=torch.bool, device="cuda").triu(1)
    decay = torch.exp((log[..., :, None] - log[..., None, :]).masked_fill(later, -math.inf)).float()
    xh, bg, cg = xs.permute(0, 1, 3, 2, 4), bs.permute(0, 1, 3, 2, 4), cs.permute(0, 1, 3, 2, 4)
    scores = (cg @ bg.transpose(-1, -2).contiguous()).repeat_interleave(share, 2)
    ahead = step.permute(0, 1, 3, 2)
    y = (scores * decay * ahead[..., None, :]) @ xh.contiguous()
    # The chunks' own states, then the state before each chunk and after the last.
    last = torch.exp(log[..., -1:] - log).float() * ahead
    bh = bg.repeat_interleave(share, 2)
    states = (xh * last[..., None]).transpose(-1, -2).contiguous() @ bh.contiguous()
    ends = torch.cumsum(log[..., -1], 1)  # (seqs, chunks, heads)
    before = torch.cat([torch.zeros_like(ends[:, :1]), ends], 1).permute(0, 2, 1)  # (seqs, heads, chunks + 1)
    gone = torch.ones(chunks + 1, chunks, dtype=torch.bool, device="cuda").triu(0)
    join = torch.exp((before[..., :, None] - before[..., None, 1:]).masked_fill(gone, -math.inf)).float()
    flat = states.permute(0, 2, 1, 3, 4).reshape(seqs, heads, chunks, dim * width)
    held = join @ flat.contiguous()
    if start is not None:
        held = held + torch.exp(before).float()[..., None] * start.reshape(seqs, heads, 1, dim * width)
    held = held.reshape(seqs, heads, chunks + 1, dim, width)
    ch = cg.repeat_interleave(share, 2)
    y = y + torch.exp(log).float()[..., None] * (ch @ held[:, :, :-1].permute(0, 2, 1, 4, 3).contiguous())
    y = y + D[:, None, None] * xh
    y = y.permute(0, 1, 3, 2, 4).reshape(seqs * total, heads, dim)
    return y[_places(offsets, tokens, total)], held[:, :, -1]


def _conv_plain(x, weight, bias, offsets, start, length):
    tokens, channels = x.shape
    taps = weight.shape[1]
    at, valid, total = _rows(offsets, length, 1)
    rows = _unpack(x, at, valid)
    head = rows.new_zeros(rows.shape[0], taps - 1, channels) if start is None else start
    rows = torch.cat([head, rows], 1)
    y = sum(rows[:, k:k + total] * weight[:, k] for k in range(taps)) + bias
    y = F.silu(y).reshape(-1, channels)[_places(offsets, tokens, total)]
    ends = (offsets[1:] - offsets[:-1]).long()[:, None] + torch.arange(taps - 1, device="cuda")
    return y, torch.gather(rows, 1, ends[..., None].expand(-1, -1, channels))


def _rms(v, weight):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * weight


def _norms_plain(residual, out, gate, post, scale, pre):
    if out is not None:
        residual = residual + scale * _rms(out if gate is None else out * F.silu(gate), post)
    return residual, None if pre is None else _rms(residual, pre)


def _f32(*tensors):
    return [None if t is None else t.float() for t in tensors]


def _gradients(function, inputs, given):
    """The gradients of sum(outputs * given) at the inputs, in 32 bits (None where there is none)."""
    with torch.enable_grad():
        leaves = [None if t is None else t.float().detach().requires_grad_() for t in inputs]
        pairs = [(o, g.float()) for o, g in zip(function(*leaves), given) if o is not None and g is not None]
        wanted = [t for t in leaves if t is not None]
        got = iter(torch.autograd.grad([o for o, _ in pairs], wanted, [g for _, g in pairs]))
    return [None if t is None else next(got).to(t.dtype) for t in inputs]


# ---------------------------------------------------------------------------------------------
# One pass.


def run(state):
    return globals()["_run_" + state["op"]](state)


def _run_scan(s):
    if own:
        from uor_fbs import trunk
        y, final = trunk.scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], dt_bias=s["dt_bias"],
                              offsets=s["offsets"], initial=s["start"])
        return dict(y=y, final=final)
    x, dt, B, C = _f32(s["x"], s["dt"], s["B"], s["C"])
    y, final = _scan_plain(x, dt, s["A"], B, C, s["D"], s["dt_bias"], s["offsets"], s["start"], s["length"])
    return dict(y=y.to(s["x"].dtype), final=final)


SCAN_GRADS = ("dx", "ddt", "dA", "dB", "dC", "dD", "ddt_bias", "dinitial")


def _run_scan_grad(s):
    if own:
        from uor_fbs import trunk
        got = trunk.scan_backward(s["dy"], s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], dt_bias=s["dt_bias"],
                                  offsets=s["offsets"], initial=s["start"], dfinal=s["d_final"])
        return {k: getattr(got, k) for k in SCAN_GRADS}
    got = _gradients(lambda *v: _scan_plain(*v[:7], s["offsets"], v[7], s["length"]),
                     [s[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "start")], (s["dy"], s["d_final"]))
    return dict(zip(SCAN_GRADS, got))


def _run_scan_step(s):
    if own:
        from uor_fbs import trunk
        y = trunk.scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["held"], slots=s["index"], D=s["D"],
                            dt_bias=s["dt_bias"])
        return dict(y=y, held=s["held"])
    x, dt, B, C = _f32(s["x"], s["dt"], s["B"], s["C"])
    share = s["heads"] // s["groups"]
    step, at = F.softplus(dt + s["dt_bias"]), s["index"].long()
    h = s["held"][at] * torch.exp(step * s["A"])[..., None, None]
    h = h + (step[..., None] * x)[..., None] * B.repeat_interleave(share, 1)[:, :, None, :]
    s["held"][at] = h
    y = (h * C.repeat_interleave(share, 1)[:, :, None, :]).sum(-1) + s["D"][:, None] * x
    return dict(y=y.to(s["x"].dtype), held=s["held"])


def _run_conv(s):
    if own:
        from uor_fbs import trunk
        y, final = trunk.conv(s["x"], s["weight"], s["bias"], offsets=s["offsets"], initial=s["start"])
        return dict(y=y, final=final)
    x, start = _f32(s["x"], s["start"])
    y, final = _conv_plain(x, s["weight"], s["bias"], s["offsets"], start, s["length"])
    return dict(y=y.to(s["x"].dtype), final=final.to(s["x"].dtype))


CONV_GRADS = ("dx", "dweight", "dbias", "dinitial")


def _run_conv_grad(s):
    if own:
        from uor_fbs import trunk
        got = trunk.conv_backward(s["dy"], s["x"], s["weight"], s["bias"], offsets=s["offsets"],
                                  initial=s["start"], dfinal=s["d_final"])
        return {k: getattr(got, k) for k in CONV_GRADS}
    got = _gradients(lambda x, w, b, start: _conv_plain(x, w, b, s["offsets"], start, s["length"]),
                     [s["x"], s["weight"], s["bias"], s["start"]], (s["dy"], s["d_final"]))
    return dict(zip(CONV_GRADS, got))


def _run_conv_step(s):
    if own:
        from uor_fbs import trunk
        y = trunk.conv_step(s["x"], s["weight"], s["held"], s["bias"], slots=s["index"])
        return dict(y=y, held=s["held"])
    at = s["index"].long()
    rows = torch.cat([s["held"][at], s["x"][:, None]], 1)
    y = F.silu((rows.float() * s["weight"].t()).sum(1) + s["bias"])
    s["held"][at] = rows[:, 1:]
    return dict(y=y.to(s["x"].dtype), held=s["held"])


def _run_norms(s):
    if own:
        from uor_fbs import trunk
        residual, normed = trunk.norms(s["residual"], s["out"], gate=s["gate"], post=s["post"], scale=s["scale"],
                                       pre=s["pre"], eps=EPS)
        return dict(residual=residual if s["out"] is not None else None, normed=normed)
    residual, normed = _norms_plain(*_f32(s["residual"], s["out"], s["gate"]), s["post"], s["scale"], s["pre"])
    dtype = s["residual"].dtype
    return dict(residual=residual.to(dtype) if s["out"] is not None else None,
                normed=None if normed is None else normed.to(dtype))


NORM_GRADS = ("dresidual", "dout", "dgate", "dpost", "dscale", "dpre")


def _run_norms_grad(s):
    if own:
        from uor_fbs import trunk
        got = trunk.norms_backward(s["d_residual"], s["d_normed"], s["residual"], s["out"], gate=s["gate"],
                                   post=s["post"], scale=s["scale"], pre=s["pre"], eps=EPS)
        return {k: getattr(got, k) for k in NORM_GRADS}
    got = _gradients(_norms_plain, [s[k] for k in ("residual", "out", "gate", "post", "scale", "pre")],
                     (s["d_residual"], s["d_normed"]))
    return dict(zip(NORM_GRADS, got))


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without.


def work(case):
    op, size = case["op"], 2 if case["dtype"] == "bf16" else 4
    if op.startswith("norms"):
        values = case["rows"] * case["width"]
        gate, post, pre = case["gate"], case["post"], case["pre"]
        if op == "norms":  # residual in; out, gate in and the residual out; the normed rows out
            return dict(bytes=size * values * (1 + 2 * post + gate + pre), flops=values * (8 * post + 6 * gate + 5 * pre))
        # The residual is read where its norm is differentiated, and the gradients of the rows written.
        return dict(bytes=size * values * (2 + pre * 2 + post * 2 + gate * 2),
                    flops=values * (24 * post + 12 * gate + 12 * pre))
    n = case["seqs"]
    tokens = n if op.endswith("_step") else int(_lengths(case).sum())
    grad, step = op.endswith("_grad"), op.endswith("_step")
    if op.startswith("conv"):
        c, k = case["channels"], case["taps"]
        held = n * (k - 1) * c * size * (2 if step else 1 + case["initial"] if not grad else 3 * case["initial"])
        return dict(bytes=tokens * c * size * (3 if grad else 2) + held + 4 * c * (k + 1) * (1 + grad),
                    flops=tokens * c * (6 * k + 12 if grad else 2 * k + 5))
    h, g, p, m = case["heads"], case["groups"], case["dim"], case["state"]
    held = n * h * p * m * 4 * (2 if step else 1 + case["initial"] if not grad else 3 * case["initial"])
    row = h * p * (3 if grad else 2) + (h + 2 * g * m) * (2 if grad else 1)
    return dict(bytes=tokens * row * size + held, flops=tokens * h * p * m * (13 if grad else 5))


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits, row after row.


def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"].replace("_grad", "")](s, case)


def _wide(s, *names):
    return [None if s.get(k) is None else s[k].double() for k in names]


def _sigma(v):
    return 1 / (1 + torch.exp(-v))


def _scan_rows(s):
    """Sequences longest first and, for each row, how many of them still have one."""
    offsets = s["offsets"].cpu().numpy().astype(np.int64)
    lengths = offsets[1:] - offsets[:-1]
    order = np.argsort(-lengths, kind="stable")
    return offsets, lengths, order


def _exact_scan(s, case):
    x, dt, A, B, C, D, bias, start, dy, d_final = _wide(s, "x", "dt", "A", "B", "C", "D", "dt_bias", "start", "dy", "d_final")
    grad = case["op"] == "scan_grad"
    tokens, heads, dim = x.shape
    groups, width = B.shape[1:]
    share = heads // groups
    offsets, lengths, order = _scan_rows(s)
    longest = int(lengths.max())
    most = max(1, int(4e9 // (8 * heads * dim * width * (longest if grad else 1))))  # sequences at once
    if (longest * -(-len(order) // most)) * (3 if grad else 1) > 100_000:
        return None
    raw = dt + bias
    step = torch.where(raw > 0, raw, 0.0) + torch.log1p(torch.exp(-raw.abs()))
    fade = torch.exp(step * A)
    Bh, Ch = (v[:, torch.arange(heads, device="cuda") // share] for v in (B, C))
    y = torch.zeros_like(x)
    final = torch.zeros(len(order), heads, dim, width, dtype=torch.float64, device="cuda")
    if grad:
        dx, dstep, da = torch.zeros_like(x), torch.zeros_like(dt), torch.zeros_like(dt)
        dBh, dCh, dstart = torch.zeros_like(Bh), torch.zeros_like(Ch), torch.zeros_like(final)
    for first in range(0, len(order), most):
        part = order[first:first + most]
        seq = torch.from_numpy(part).cuda()
        base, size = torch.from_numpy(offsets[part]).cuda(), lengths[part]
        h = torch.zeros_like(final[seq]) if start is None else start[seq]
        past = []
        for t in range(int(size.max(initial=0))):
            n = int((size > t).sum())
            r = base[:n] + t
            if grad:
                past.append(h[:n].clone())
            h[:n] = h[:n] * fade[r][..., None, None] + (step[r][..., None] * x[r])[..., None] * Bh[r][:, :, None, :]
            y[r] = (h[:n] @ Ch[r][..., None])[..., 0] + D[:, None] * x[r]
        final[seq] = h
        if not grad:
            continue
        d = torch.zeros_like(h) if d_final is None else d_final[seq].clone()
        for t in range(int(size.max(initial=0)) - 1, -1, -1):
            n = int((size > t).sum())
            r, d_now = base[:n] + t, d[:n]
            f, old = fade[r][..., None, None], past.pop()
            new = f * old + (step[r][..., None] * x[r])[..., None] * Bh[r][:, :, None, :]
            d_now = d_now + dy[r][..., None] * Ch[r][:, :, None, :]
            dCh[r] = (dy[r][:, :, None] @ new)[:, :, 0]
            into = (d_now @ Bh[r][..., None])[..., 0]
            dx[r] = step[r][..., None] * into + D[:, None] * dy[r]
            dBh[r] = step[r][..., None] * (x[r][:, :, None] @ d_now)[:, :, 0]
            da[r] = (d_now * old * f).sum((-1, -2))
            dstep[r] = (x[r] * into).sum(-1) + A * da[r]
            d[:n] = d_now * f
        dstart[seq] = d
    if not grad:
        return dict(y=y, final=final)
    draw_ = dstep * _sigma(raw)
    join = lambda v: v.reshape(tokens, groups, share, width).sum(2)  # noqa: E731
    return dict(dx=dx, ddt=draw_, dA=(da * step).sum(0), dB=join(dBh), dC=join(dCh), dD=(dy * x).sum((0, 2)),
                ddt_bias=draw_.sum(0), dinitial=None if start is None else dstart)


def _exact_scan_step(s, case):
    x, dt, A, B, C, D, bias, held = _wide(s, "x", "dt", "A", "B", "C", "D", "dt_bias", "held")
    raw, at = dt + bias, s["index"].long()
    step = torch.where(raw > 0, raw, 0.0) + torch.log1p(torch.exp(-raw.abs()))
    group = torch.arange(case["heads"], device="cuda") // (case["heads"] // case["groups"])
    held[at] = held[at] * torch.exp(step * A)[..., None, None] + (x * step[..., None])[..., None] * B[:, group][:, :, None, :]
    return dict(y=(held[at] @ C[:, group][..., None])[..., 0] + x * D[:, None], held=held)


def _exact_conv(s, case):
    x, weight, bias, start, dy, d_final = _wide(s, "x", "weight", "bias", "start", "dy", "d_final")
    taps, offsets = weight.shape[1], s["offsets"].cpu().numpy()
    seqs = len(offsets) - 1
    if start is None:
        start = x.new_zeros(seqs, taps - 1, x.shape[1])
    # The sequences one after another, each behind its taps - 1 rows of the past.
    lead = np.repeat(np.arange(1, seqs + 1), offsets[1:] - offsets[:-1]) * (taps - 1)
    here = torch.from_numpy(np.arange(x.shape[0]) + lead).cuda()
    rows = x.new_zeros(x.shape[0] + seqs * (taps - 1), x.shape[1])
    past = torch.from_numpy((offsets[:-1] + np.arange(seqs) * (taps - 1))[:, None] + np.arange(taps - 1)).cuda()
    ends = torch.from_numpy((offsets[1:] + np.arange(seqs) * (taps - 1))[:, None] + np.arange(taps - 1)).cuda()
    rows[past], rows[here] = start, x
    pre = bias.expand_as(x).clone()
    for k in range(taps):
        pre += weight[:, k] * rows[here - (taps - 1) + k]
    if case["op"] == "conv":
        return dict(y=pre * _sigma(pre), final=rows[ends])
    sig = _sigma(pre)
    d = dy * sig * (1 + pre * (1 - sig))
    drows, dweight = torch.zeros_like(rows), torch.zeros_like(weight)
    for k in range(taps):
        drows[here - (taps - 1) + k] += d * weight[:, k]
        dweight[:, k] = (d * rows[here - (taps - 1) + k]).sum(0)
    if d_final is not None:
        drows.index_put_((ends,), d_final, accumulate=True)
    return dict(dx=drows[here], dweight=dweight, dbias=d.sum(0), dinitial=drows[past] if case["initial"] else None)


def _exact_conv_step(s, case):
    x, weight, bias, held = _wide(s, "x", "weight", "bias", "held")
    at = s["index"].long()
    pre = x * weight[:, -1] + bias
    for k in range(weight.shape[1] - 1):
        pre += held[at, k] * weight[:, k]
    held[at] = torch.cat([held[at][:, 1:], x[:, None]], 1)
    return dict(y=pre * _sigma(pre), held=held)


def _exact_norms(s, case):
    r, u, z, post, scale, pre, d_residual, d_normed = _wide(
        s, "residual", "out", "gate", "post", "scale", "pre", "d_residual", "d_normed")
    inv = lambda v: 1 / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + EPS)  # noqa: E731
    if u is not None:
        act = 1.0 if z is None else z * _sigma(z)
        v = u * act
        i = inv(v)
        p = v * i * post
        r = r + scale * p
    j = inv(r)
    if case["op"] == "norms":
        return dict(residual=r if u is not None else None, normed=None if pre is None else r * j * pre)
    got = dict.fromkeys(NORM_GRADS)
    d = d_residual
    if pre is not None:
        got["dpre"] = (d_normed * r * j).sum(0)
        e = d_normed * pre
        d = d + j * e - r * j ** 3 * (e * r).mean(-1, keepdim=True)
    got["dresidual"] = d
    if u is not None:
        got["dscale"], got["dpost"] = (d * p).sum(0), (d * scale * v * i).sum(0)
        e = d * scale * post
        dv = i * e - v * i ** 3 * (e * v).mean(-1, keepdim=True)
        got["dout"] = dv * act
        if z is not None:
            sig = _sigma(z)
            got["dgate"] = dv * u * sig * (1 + z * (1 - sig))
    return got
