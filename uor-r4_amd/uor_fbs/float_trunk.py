"""A small float trunk from the operators of uor_fbs.trunk: prompts, single tokens over device slots,
and a training step, as a program would call them together.

A layer takes the normed residual n of its rows and computes

    x, B, C, dt = n W_in          x, B and C through the short convolution and silu
    y           = scan(x, dt, A, B, C)
    residual'   = residual + scale rms((y W_out) silu(n W_gate)) post,  n' = rms(residual') pre

with W_* products of torch. ``python -m uor_fbs.float_trunk`` trains one to repeat its prompts and then
lets sessions go on from them token by token.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import trunk


class Config(NamedTuple):
    vocab: int = 64
    width: int = 64
    layers: int = 2
    heads: int = 4
    groups: int = 1
    dim: int = 32
    state: int = 32
    taps: int = 4
    dtype: torch.dtype = torch.bfloat16

    @property
    def inner(self):
        return self.heads * self.dim

    @property
    def channels(self):
        return self.inner + 2 * self.groups * self.state


LAYER = ("w_in", "conv", "conv_bias", "dt_bias", "A_log", "D", "w_gate", "w_out", "post", "scale", "pre")


def make_params(cfg, seed=0, device="cuda"):
    """{name: float32 tensor}; the matrices are used in the trunk's type."""
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape, scale: (torch.randn(shape, generator=g) * scale).to(device)  # noqa: E731
    ones = lambda n, v=1.0: torch.full((n,), v, device=device)  # noqa: E731
    p = {"embed": normal(cfg.vocab, cfg.width, scale=1.0), "first": ones(cfg.width),
         "head": normal(cfg.width, cfg.vocab, scale=cfg.width ** -0.5)}
    for i in range(cfg.layers):
        layer = dict(w_in=normal(cfg.width, cfg.channels + cfg.heads, scale=cfg.width ** -0.5),
                     conv=normal(cfg.channels, cfg.taps, scale=0.5), conv_bias=ones(cfg.channels, 0.0),
                     dt_bias=ones(cfg.heads, -1.0), A_log=torch.linspace(-2.0, 1.0, cfg.heads).to(device), D=ones(cfg.heads),
                     w_gate=normal(cfg.width, cfg.width, scale=cfg.width ** -0.5),
                     w_out=normal(cfg.inner, cfg.width, scale=cfg.inner ** -0.5),
                     post=ones(cfg.width), scale=ones(cfg.width, 0.5), pre=ones(cfg.width))
        p.update({f"{i}.{k}": v for k, v in layer.items()})
    return p


def _layer(cfg, p, i):
    """The layer's parameters by name, its matrices in the trunk's type, and A."""
    w = {k: p[f"{i}.{k}"] for k in LAYER}
    for k in ("w_in", "w_gate", "w_out"):
        w[k] = w[k].to(cfg.dtype)
    w["A"] = -torch.exp(w["A_log"])
    return w


def _parts(cfg, rows):
    """x, B and C of rows after the convolution, as views."""
    gn = cfg.groups * cfg.state
    x, B, C = rows.split([cfg.inner, gn, gn], 1)
    return x.unflatten(1, (cfg.heads, cfg.dim)), B.unflatten(1, (cfg.groups, cfg.state)), C.unflatten(1, (cfg.groups, cfg.state))


class State(NamedTuple):
    """Sessions' states, a slot each: per layer the convolution's last rows and the scan's state."""
    conv: list
    scan: list


def make_state(cfg, slots, device="cuda"):
    return State([torch.zeros(slots, cfg.taps - 1, cfg.channels, dtype=cfg.dtype, device=device) for _ in range(cfg.layers)],
                 [torch.zeros(slots, cfg.heads, cfg.dim, cfg.state, device=device) for _ in range(cfg.layers)])


def prompts(cfg, p, tokens, offsets, state=None, slots=None, saved=None):
    """Logits (rows, vocab) of packed prompts. With ``state`` and ``slots`` (int64, one a prompt) the
    prompts' final states are put into their slots; ``saved`` (a list) takes what the gradients need."""
    residual = p["embed"].to(cfg.dtype)[tokens]
    _, n = trunk.norms(residual, pre=p["first"])
    for i in range(cfg.layers):
        w = _layer(cfg, p, i)
        rows = n @ w["w_in"]
        mixed, last = trunk.conv(rows[:, :cfg.channels], w["conv"], w["conv_bias"], offsets=offsets)
        x, B, C = _parts(cfg, mixed)
        y, final = trunk.scan(x, rows[:, cfg.channels:], w["A"], B, C, D=w["D"], dt_bias=w["dt_bias"], offsets=offsets)
        out, gate = y.flatten(1) @ w["w_out"], n @ w["w_gate"]
        if saved is not None:
            saved.append((residual, n, rows, mixed, y, out, gate))
        if state is not None:
            state.conv[i][slots], state.scan[i][slots] = last, final
        residual, n = trunk.norms(residual, out, gate=gate, post=w["post"], scale=w["scale"], pre=w["pre"])
    if saved is not None:
        saved.append(n)
    return (n @ p["head"].to(cfg.dtype)).float()


def step(cfg, p, tokens, state, slots):
    """Logits (rows, vocab) of one more token of each session; ``slots`` (int32) says where it lives."""
    residual = p["embed"].to(cfg.dtype)[tokens]
    _, n = trunk.norms(residual, pre=p["first"])
    for i in range(cfg.layers):
        w = _layer(cfg, p, i)
        rows = n @ w["w_in"]
        mixed = trunk.conv_step(rows[:, :cfg.channels], w["conv"], state.conv[i], w["conv_bias"], slots=slots)
        x, B, C = _parts(cfg, mixed)
        y = trunk.scan_step(x, rows[:, cfg.channels:], w["A"], B, C, state.scan[i], slots=slots, D=w["D"], dt_bias=w["dt_bias"])
        residual, n = trunk.norms(residual, y.flatten(1) @ w["w_out"], gate=n @ w["w_gate"], post=w["post"], scale=w["scale"],
                                  pre=w["pre"])
    return (n @ p["head"].to(cfg.dtype)).float()


def gradients(cfg, p, tokens, targets, offsets):
    """(loss, {name: gradient}): the mean cross entropy of the rows' next tokens (target -1: none)."""
    saved = []
    logits = prompts(cfg, p, tokens, offsets, saved=saved)
    wanted = targets >= 0
    count = wanted.sum().clamp(min=1)
    log = torch.log_softmax(logits, 1)
    at = targets.clamp(min=0)[:, None]
    loss = -(log.gather(1, at)[:, 0] * wanted).sum() / count
    d_logits = torch.exp(log)
    d_logits.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    d_logits = (d_logits * (wanted / count)[:, None]).to(cfg.dtype)

    grads = {"head": saved[-1].t().float() @ d_logits.float()}
    d_n, d_residual = d_logits @ p["head"].to(cfg.dtype).t(), None
    for i in reversed(range(cfg.layers)):
        w = _layer(cfg, p, i)
        residual, n, rows, mixed, y, out, gate = saved[i]
        d_residual = torch.zeros_like(residual) if d_residual is None else d_residual
        g = trunk.norms_backward(d_residual, d_n, residual, out, gate=gate, post=w["post"], scale=w["scale"], pre=w["pre"])
        d_residual = g.dresidual
        d_y = (g.dout @ w["w_out"].t()).unflatten(1, (cfg.heads, cfg.dim))
        x, B, C = _parts(cfg, mixed)
        s = trunk.scan_backward(d_y, x, rows[:, cfg.channels:], w["A"], B, C, D=w["D"], dt_bias=w["dt_bias"], offsets=offsets)
        d_mixed = torch.cat([s.dx.flatten(1), s.dB.flatten(1), s.dC.flatten(1)], 1)
        c = trunk.conv_backward(d_mixed, rows[:, :cfg.channels], w["conv"], w["conv_bias"], offsets=offsets)
        d_rows = torch.cat([c.dx, s.ddt], 1)
        d_n = d_rows @ w["w_in"].t() + g.dgate @ w["w_gate"].t()
        layer = dict(w_in=n.t().float() @ d_rows.float(), conv=c.dweight, conv_bias=c.dbias, dt_bias=s.ddt_bias, A_log=s.dA * w["A"],
                     D=s.dD, w_gate=n.t().float() @ g.dgate.float(), w_out=y.flatten(1).t().float() @ g.dout.float(),
                     post=g.dpost, scale=g.dscale, pre=g.dpre)
        grads.update({f"{i}.{k}": v for k, v in layer.items()})
    first = trunk.norms_backward(d_residual, d_n, saved[0][0], pre=p["first"])
    grads["first"] = first.dpre
    grads["embed"] = torch.zeros_like(p["embed"]).index_add_(0, tokens, first.dresidual.float())
    return loss, grads


def repeats(cfg, count, length, generator, device="cuda"):
    """(tokens, targets, offsets): prompts that say ``length`` random tokens twice; only the second
    time has targets."""
    said = torch.randint(1, cfg.vocab, (count, length), generator=generator)
    rows = torch.cat([said, torch.zeros(count, 1, dtype=torch.long), said], 1)
    targets = torch.full_like(rows, -1)
    targets[:, length:-1] = rows[:, length + 1:]
    offsets = torch.arange(count + 1, dtype=torch.int32) * rows.shape[1]
    return rows.flatten().to(device), targets.flatten().to(device), offsets.to(device)


def train(cfg, p, steps, count=64, length=8, rate=3e-3, seed=1, report=None):
    """``steps`` steps of Adam on ``repeats``; the losses."""
    g = torch.Generator().manual_seed(seed)
    m, v = ({k: torch.zeros_like(t) for k, t in p.items()} for _ in range(2))
    losses = []
    for n in range(1, steps + 1):
        loss, grads = gradients(cfg, p, *repeats(cfg, count, length, g, p["embed"].device))
        for k, t in p.items():
            m[k].lerp_(grads[k], 0.1)
            v[k].lerp_(grads[k].square(), 0.01)
            t.sub_(rate * (m[k] / (1 - 0.9 ** n)) / ((v[k] / (1 - 0.99 ** n)).sqrt() + 1e-8))
        losses.append(loss)
        if report and n % report == 0:
            print(f"step {n}: loss {loss.item():.3f}", flush=True)
    return [loss.item() for loss in losses]


def reply(cfg, p, tokens, offsets, count, state, slots):
    """``count`` greedy tokens of each prompt's session, (prompts, count). A prompt has a token at least."""
    if bool((offsets[1:] <= offsets[:-1]).any()):
        raise ValueError("a prompt of no tokens has nothing that a reply could follow")
    logits = prompts(cfg, p, tokens, offsets, state, slots.long())
    now = logits[offsets[1:].long() - 1].argmax(1)
    said = [now]
    for _ in range(count - 1):
        now = step(cfg, p, now, state, slots).argmax(1)
        said.append(now)
    return torch.stack(said, 1)


def main():
    cfg, length = Config(), 8
    p = make_params(cfg)
    train(cfg, p, 400, length=length, report=50)
    tokens, _, _ = repeats(cfg, 32, length, torch.Generator().manual_seed(99))
    rows = tokens.view(32, -1)[:, :length + 1]
    offsets = torch.arange(33, dtype=torch.int32, device=rows.device) * (length + 1)
    said = reply(cfg, p, rows.flatten(), offsets, length, make_state(cfg, 40), torch.arange(39, 7, -1, dtype=torch.int32, device=rows.device))
    print(f"repeated {(said == rows[:, :length]).float().mean().item():.1%} of the tokens of 32 new prompts")


if __name__ == "__main__":
    main()
