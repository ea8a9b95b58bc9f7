"""The float trunk's operators from their definitions, in 64 bits on the CPU, row after row: the
oracle of uor_fbs.trunk. Each gradient is the formula's; test_trunk_oracle.py holds it to central
differences. With `magnitude` the same sums run over absolute values: what rounding is relative to.
"""

import numpy as np
import torch

F64 = torch.float64


def offsets_of(lengths):
    off = np.zeros(len(lengths) + 1, np.int32)
    off[1:] = np.cumsum(lengths)
    return torch.from_numpy(off)


def wide(*tensors):
    return [None if t is None else t.detach().cpu().to(F64) for t in tensors]


def softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def bounds(offsets, rows):
    if offsets is None:
        return [(0, rows)]
    off = [min(max(int(v), 0), rows) for v in offsets.tolist()]
    return [(a, max(a, b)) for a, b in zip(off, off[1:])]


def scan(x, dt, A, B, C, D=None, dt_bias=None, offsets=None, initial=None, magnitude=False):
    x, dt, A, B, C, D, dt_bias, initial = wide(x, dt, A, B, C, D, dt_bias, initial)
    rows, heads, dim = x.shape
    share = heads // B.shape[1]
    step = softplus(dt + (0 if dt_bias is None else dt_bias))
    decay = torch.exp(step * A)
    if magnitude:
        x, B, C = x.abs(), B.abs(), C.abs()
        D, initial = (None if t is None else t.abs() for t in (D, initial))
    B, C = B.repeat_interleave(share, 1), C.repeat_interleave(share, 1)
    spans = bounds(offsets, rows)
    y = torch.zeros_like(x)
    final = torch.zeros(len(spans), heads, dim, B.shape[2], dtype=F64)
    for s, (a, b) in enumerate(spans):
        h = final[s].clone() if initial is None else initial[s].clone()
        for t in range(a, b):
            h = h * decay[t][:, None, None] + (step[t][:, None] * x[t])[:, :, None] * B[t][:, None, :]
            y[t] = (h * C[t][:, None, :]).sum(-1) + (0 if D is None else D[:, None] * x[t])
        final[s] = h
    return y, final


def scan_backward(dy, x, dt, A, B, C, D=None, dt_bias=None, offsets=None, initial=None, dfinal=None, magnitude=False):
    """A dict of the gradients, with `q`: C_t . (h_t^T dy_t) of each row and head."""
    dy, x, dt, A, B, C, D, dt_bias, initial, dfinal = wide(dy, x, dt, A, B, C, D, dt_bias, initial, dfinal)
    rows, heads, dim = x.shape
    groups, state = B.shape[1:]
    share = heads // groups
    raw = dt + (0 if dt_bias is None else dt_bias)
    step = softplus(raw)
    decay = torch.exp(step * A)
    if magnitude:
        dy, x, B, C = dy.abs(), x.abs(), B.abs(), C.abs()
        A = A.abs()
        D, initial, dfinal = (None if t is None else t.abs() for t in (D, initial, dfinal))
    Bh, Ch = B.repeat_interleave(share, 1), C.repeat_interleave(share, 1)
    spans = bounds(offsets, rows)
    dx, da, dstep = torch.zeros_like(x), torch.zeros_like(dt), torch.zeros_like(dt)
    dB, dC, q = torch.zeros_like(Bh), torch.zeros_like(Ch), torch.zeros_like(dt)
    dinitial = torch.zeros(len(spans), heads, dim, state, dtype=F64)
    for s, (a, b) in enumerate(spans):
        h = torch.zeros(heads, dim, state, dtype=F64) if initial is None else initial[s]
        past = []
        for t in range(a, b):
            past.append(h)
            h = h * decay[t][:, None, None] + (step[t][:, None] * x[t])[:, :, None] * Bh[t][:, None, :]
        g = torch.zeros_like(h) if dfinal is None else dfinal[s]
        for t in range(b - 1, a - 1, -1):
            g = g + dy[t][:, :, None] * Ch[t][:, None, :]
            dC[t] = (dy[t][:, :, None] * h).sum(1)
            q[t] = (dC[t] * Ch[t]).sum(-1)
            into = (g * Bh[t][:, None, :]).sum(-1)
            dx[t] = step[t][:, None] * into + (0 if D is None else D[:, None] * dy[t])
            dB[t] = step[t][:, None] * (x[t][:, :, None] * g).sum(1)
            h = past.pop()
            da[t] = decay[t] * (g * h).sum((1, 2))
            dstep[t] = (x[t] * into).sum(-1) + A * da[t]
            g = g * decay[t][:, None, None]
        dinitial[s] = g
    sigma = 1 / (1 + torch.exp(-raw))
    return dict(dx=dx, ddt=dstep * sigma, dA=(da * step).sum(0), dB=dB.reshape(rows, groups, share, state).sum(2),
                dC=dC.reshape(rows, groups, share, state).sum(2), dD=None if D is None else (dy * x).sum((0, 2)),
                ddt_bias=None if dt_bias is None else (dstep * sigma).sum(0),
                dinitial=None if initial is None else dinitial, q=q, step=step)


def scan_step(x, dt, A, B, C, states, index, D=None, dt_bias=None, magnitude=False):
    """(y, states): rows whose index is outside are skipped."""
    states = wide(states)[0].clone()
    if magnitude:
        states = states.abs()
    y = torch.zeros(x.shape, dtype=F64)
    for i, slot in enumerate(range(x.shape[0]) if index is None else index.tolist()):
        if 0 <= slot < states.shape[0]:
            row = [v[i:i + 1] for v in (x, dt, B, C)]
            y[i:i + 1], states[slot:slot + 1] = scan(row[0], row[1], A, row[2], row[3], D, dt_bias,
                                                     initial=states[slot:slot + 1], magnitude=magnitude)
    return y, states


def conv(x, weight, bias=None, offsets=None, initial=None, silu=True, magnitude=False):
    """(y, final, the values before the activation's magnitude)"""
    x, weight, bias, initial = wide(x, weight, bias, initial)
    taps, channels = weight.shape[1], x.shape[1]
    spans = bounds(offsets, x.shape[0])
    y, size = torch.zeros_like(x), torch.zeros_like(x)
    final = torch.zeros(len(spans), taps - 1, channels, dtype=F64)
    for s, (a, b) in enumerate(spans):
        rows = torch.cat([final[s] if initial is None else initial[s], x[a:b]])
        for t in range(b - a):
            y[a + t] = (rows[t:t + taps] * weight.t()).sum(0) + (0 if bias is None else bias)
            size[a + t] = (rows[t:t + taps] * weight.t()).abs().sum(0) + (0 if bias is None else bias.abs())
        final[s] = rows[rows.shape[0] - (taps - 1):]
    return y / (1 + torch.exp(-y)) if silu else y, final, size


def conv_backward(dy, x, weight, bias=None, offsets=None, initial=None, dfinal=None, silu=True):
    """(gradients, their sums of absolute terms), as dicts."""
    dy, x, weight, bias, initial, dfinal = wide(dy, x, weight, bias, initial, dfinal)
    taps, channels = weight.shape[1], x.shape[1]
    spans = bounds(offsets, x.shape[0])
    zeros = lambda *s: torch.zeros(*s, dtype=F64)  # noqa: E731
    got = [dict(dx=zeros(*x.shape), dweight=zeros(*weight.shape), dbias=zeros(channels), dinitial=zeros(len(spans), taps - 1, channels))
           for _ in range(2)]
    for s, (a, b) in enumerate(spans):
        rows = torch.cat([zeros(taps - 1, channels) if initial is None else initial[s], x[a:b]])
        drows = [zeros(*rows.shape), zeros(*rows.shape)]
        for t in range(b - a):
            d = dy[a + t]
            m = d.abs()
            if silu:
                v = (rows[t:t + taps] * weight.t()).sum(0) + (0 if bias is None else bias)
                sig = 1 / (1 + torch.exp(-v))
                d = d * sig * (1 + v * (1 - sig))
                # The slope changes by less than half of the change in v.
                size = (rows[t:t + taps] * weight.t()).abs().sum(0) + (0 if bias is None else bias.abs())
                m = m * (1 + size)
            for g, e, f in ((0, d, lambda v: v), (1, m, torch.abs)):
                for k in range(taps):
                    drows[g][t + k] += e * f(weight[:, k])
                    got[g]["dweight"][:, k] += e * f(rows[t + k])
                got[g]["dbias"] += e
        for g, f in ((0, lambda v: v), (1, torch.abs)):
            if dfinal is not None:
                drows[g][b - a:] += f(dfinal[s])
            got[g]["dinitial"][s], got[g]["dx"][a:b] = drows[g][:taps - 1], drows[g][taps - 1:]
    return got


def norms(residual, out=None, gate=None, post=None, scale=None, pre=None, eps=1e-6):
    residual, out, gate, post, scale, pre = wide(residual, out, gate, post, scale, pre)
    r = 0 if residual is None else residual
    if out is not None:
        v = out if gate is None else out * gate / (1 + torch.exp(-gate))
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
        r = r + (1 if scale is None else scale) * v * (1 if post is None else post)
    return r, None if pre is None else r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps) * pre


def norms_backward(dresidual_out, dnormed, residual, out=None, gate=None, post=None, scale=None, pre=None, eps=1e-6):
    """(gradients, their sums of absolute terms), as dicts (None where there is no input)."""
    dr, dn, residual, out, gate, post, scale, pre = wide(dresidual_out, dnormed, residual, out, gate, post, scale, pre)
    like = out if residual is None else residual
    one = torch.ones(like.shape[1], dtype=F64)
    got, size = ({k: None for k in ("dresidual", "dout", "dgate", "dpost", "dscale", "dpre")} for _ in range(2))
    r, _ = norms(residual, out, gate, post, scale, None, eps)
    # r' is a sum itself: the sum of absolute terms is its two parts'.
    rm = r.abs() if out is None or residual is None else residual.abs() + (r - residual).abs()
    d = torch.zeros_like(like) if dr is None else dr
    m = d.abs()
    if pre is not None:
        j = 1 / torch.sqrt((r * r).mean(-1, keepdim=True) + eps)
        e = torch.zeros_like(d) if dn is None else dn * pre
        got["dpre"] = torch.zeros_like(one) if dn is None else (dn * r * j).sum(0)
        size["dpre"] = torch.zeros_like(one) if dn is None else ((dn * j).abs() * rm).sum(0)
        d = d + j * e - r * j ** 3 * (e * r).mean(-1, keepdim=True)
        m = m + (j * e).abs() + rm * j ** 3 * (e.abs() * rm).mean(-1, keepdim=True)
    if residual is not None:
        got["dresidual"], size["dresidual"] = d, m
    if out is None:
        return got, size
    sig = None if gate is None else 1 / (1 + torch.exp(-gate))
    act = 1 if gate is None else gate * sig
    post_, scale_ = (one if p is None else p for p in (post, scale))
    v = out * act
    i = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    for store, t, f in ((got, d, lambda x: x), (size, m, torch.abs)):
        if post is not None:
            store["dpost"] = (t * f(scale_ * v * i)).sum(0)
        if scale is not None:
            store["dscale"] = (t * f(post_ * v * i)).sum(0)
    e, em = d * scale_ * post_, m * (scale_ * post_).abs()
    dv = i * e - v * i ** 3 * (e * v).mean(-1, keepdim=True)
    dvm = i * em + v.abs() * i ** 3 * (em * v.abs()).mean(-1, keepdim=True)
    got["dout"], size["dout"] = dv * act, dvm * (1 if gate is None else act.abs())
    if gate is not None:
        slope = sig * (1 + gate * (1 - sig))
        got["dgate"], size["dgate"] = dv * out * slope, dvm * out.abs() * sig * (1 + gate.abs() * (1 - sig))
    return got, size
