"""A small float trunk from the operators of uor_fbs.trunk: prompts, single tokens over device slots,
and a training step, as a program would call them together.

A layer takes the normed residual n of its rows and computes

    x, B, C, dt = n W_in          x, B and C through the short convolution and silu
    y           = scan(x, dt, A, B, C)
    residual'   = residual + scale rms((y W_out) silu(n W_gate)) post,  n' = rms(residual') pre

with W_* products of torch. Its rows begin as the embedding's and end at the head over the vocabulary: as logits,
or (``Config.keep_logits`` false) as a loss, its gradients and a choice of tokens that keep none. A token or target
outside the vocabulary (not the last words by negative numbers) is none: its row begins as zeros.
``python -m uor_fbs.float_trunk`` trains one to repeat its prompts and then lets sessions go on from them
token by token.
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
    keep_logits: bool = True  # the loss, its gradients and replies from whole logits of the trunk's type

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


def _logits(cfg, p, n):
    return (n @ p["head"].to(cfg.dtype)).float()


def _words(cfg, p):
    """The head's matrix, a row a word."""
    return p["head"].t().to(cfg.dtype, memory_format=torch.contiguous_format)


def _embed(cfg, p, tokens):
    """The tokens' rows. The table may be of any floating type, the tokens on another device, and both of more words and rows
    than one lookup takes: a word is none for the other parts of the table, whose rows are zeros then."""
    table = p["embed"] if p["embed"].dtype in trunk.DTYPES else p["embed"].to(cfg.dtype)
    tokens = tokens.to(table.device)
    if tokens.numel() <= trunk.MAX_ROWS and len(table) <= trunk.MAX_VOCAB:
        return trunk.embed(tokens, table, dtype=cfg.dtype)
    words = range(0, len(table), trunk.MAX_VOCAB)
    return torch.cat([sum(trunk.embed(some - at, table[at:at + trunk.MAX_VOCAB], dtype=cfg.dtype) for at in words)
                      for some in tokens.long().split(trunk.MAX_ROWS)])


def _embed_backward(p, d_rows, tokens):
    """The table's gradient."""
    table, tokens = p["embed"], tokens.to(p["embed"].device)
    if tokens.numel() <= trunk.MAX_ROWS and len(table) <= trunk.MAX_VOCAB:
        return trunk.embed_backward(d_rows, tokens, table)
    parts = list(zip(d_rows.split(trunk.MAX_ROWS), tokens.long().split(trunk.MAX_ROWS)))
    return torch.cat([sum(trunk.embed_backward(d, some - at, table[at:at + trunk.MAX_VOCAB]) for d, some in parts)
                      for at in range(0, len(table), trunk.MAX_VOCAB)])


def _prompt_rows(cfg, p, tokens, offsets, state=None, slots=None, saved=None):
    """The rows before the head of packed prompts."""
    residual = _embed(cfg, p, tokens)
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
    return n


def prompts(cfg, p, tokens, offsets, state=None, slots=None, saved=None):
    """Logits (rows, vocab) of packed prompts. With ``state`` and ``slots`` (int64, one a prompt) the
    prompts' final states are put into their slots; ``saved`` (a list) takes what the gradients need."""
    return _logits(cfg, p, _prompt_rows(cfg, p, tokens, offsets, state, slots, saved))


def _step_rows(cfg, p, tokens, state, slots):
    """The rows before the head of one more token of each session."""
    residual = _embed(cfg, p, tokens)
    _, n = trunk.norms(residual, pre=p["first"])
    for i in range(cfg.layers):
        w = _layer(cfg, p, i)
        rows = n @ w["w_in"]
        mixed = trunk.conv_step(rows[:, :cfg.channels], w["conv"], state.conv[i], w["conv_bias"], slots=slots)
        x, B, C = _parts(cfg, mixed)
        y = trunk.scan_step(x, rows[:, cfg.channels:], w["A"], B, C, state.scan[i], slots=slots, D=w["D"], dt_bias=w["dt_bias"])
        residual, n = trunk.norms(residual, y.flatten(1) @ w["w_out"], gate=n @ w["w_gate"], post=w["post"], scale=w["scale"],
                                  pre=w["pre"])
    return n


def step(cfg, p, tokens, state, slots):
    """Logits (rows, vocab) of one more token of each session; ``slots`` (int32) says where it lives."""
    return _logits(cfg, p, _step_rows(cfg, p, tokens, state, slots))


def gradients(cfg, p, tokens, targets, offsets):
    """(loss, {name: gradient}): the mean cross entropy of the rows' next tokens (a target outside the vocabulary: none)."""
    saved = []
    n = _prompt_rows(cfg, p, tokens, offsets, saved=saved)
    wanted = (targets >= 0) & (targets < cfg.vocab)
    count = wanted.sum().clamp(min=1)
    if cfg.keep_logits:
        log = torch.log_softmax(_logits(cfg, p, n), 1)
        at = torch.where(wanted, targets, 0)[:, None]
        loss = -(log.gather(1, at)[:, 0] * wanted).sum() / count
        d_logits = torch.exp(log)
        d_logits.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
        d_logits = (d_logits * (wanted / count)[:, None]).to(cfg.dtype)
        grads = {"head": n.t().float() @ d_logits.float()}
        d_n = d_logits @ p["head"].to(cfg.dtype).t()
    else:
        words = _words(cfg, p)
        losses, lse = trunk.loss(n, words, targets)
        loss = losses.sum() / count
        g = trunk.loss_backward(wanted / count, n, words, targets, lse, dtype=torch.float32)
        grads, d_n = {"head": g.dweight.t()}, g.dx
    d_residual = None
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
    grads["embed"] = _embed_backward(p, first.dresidual, tokens)
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
    last = offsets[1:].long() - 1
    if cfg.keep_logits:
        now = prompts(cfg, p, tokens, offsets, state, slots.long())[last].argmax(1)
        next_of = lambda now: step(cfg, p, now, state, slots).argmax(1)  # noqa: E731
    else:
        words = _words(cfg, p)
        now, _ = trunk.choose(_prompt_rows(cfg, p, tokens, offsets, state, slots.long())[last], words)
        next_of = lambda now: trunk.choose(_step_rows(cfg, p, now, state, slots), words)[0]  # noqa: E731
    said = [now]
    for _ in range(count - 1):
        now = next_of(now)
        said.append(now)
    return torch.stack(said, 1)


def main():
    cfg, length = Config(keep_logits=False), 8
    p = make_params(cfg)
    train(cfg, p, 400, length=length, report=50)
    tokens, _, _ = repeats(cfg, 32, length, torch.Generator().manual_seed(99))
    rows = tokens.view(32, -1)[:, :length + 1]
    offsets = torch.arange(33, dtype=torch.int32, device=rows.device) * (length + 1)
    said = reply(cfg, p, rows.flatten(), offsets, length, make_state(cfg, 40), torch.arange(39, 7, -1, dtype=torch.int32, device=rows.device))
    print(f"repeated {(said == rows[:, :length]).float().mean().item():.1%} of the tokens of 32 new prompts")


if __name__ == "__main__":
    main()
