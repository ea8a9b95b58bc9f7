"""Both ends of a float trunk over its vocabulary, as cases that can be timed and compared.

A trunk that is trained or answers in floating point begins with the lookup of its tokens' rows and
ends with a product over the whole vocabulary. These are the two ends as a program needs them that
keeps no logits: the embedding's lookup and its gradient, the head's softmax cross entropy with its
gradients, and for single tokens the head's greedy choice with its log probability.

``own = False`` computes them in their plain form from elementary torch operations in 32 bits,
rounded once at the end, with the logits whole. ``own = True`` calls ``uor_fbs.trunk``.

    embed      y_t = scale E[token_t], 0 for a token outside the vocabulary (padding)
    embed_grad dE_v = scale sum of dy_t over the rows t whose token is v
    loss       z_tv = x_t . W_v, lse_t = log sum_v e^z_tv, loss_t = lse_t - z_t,target_t; a row whose
               target is outside the vocabulary (a prompt's, or padding) has neither: both are 0
    loss_grad  the same with the gradients of sum_t weight_t loss_t at x and W: a training step's end
    choose     token_t = argmax_v z_tv (the lowest of equals), logprob_t = z_t,token - lse_t
"""

from __future__ import annotations

import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "uor-r4_amd"))

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # A training step's first operator: 2,048 rows of 128 tokens, a table of 32-bit parameters
        # looked up as bf16 rows at width 256.
        dict(name="embed_w256_262144", op="embed", table="f32", dtype="bf16", rows=262144, width=256, vocab=32768,
             padding=0.0, scale=1.0),
        # The serving loop: 1,024 sessions' last tokens, from a table in the trunk's type, scaled.
        dict(name="embed_w512_b1024", op="embed", table="bf16", dtype="bf16", rows=1024, width=512, vocab=32768,
             padding=0.0, scale=22.627416998),
        # The training step's last operator: words as frequent as words are, so a few rows take a
        # large part of all gradients.
        dict(name="embed_grad_w256_262144", op="embed_grad", table="f32", dtype="bf16", rows=262144, width=256,
             vocab=32768, padding=0.0, scale=1.0),
        # A large vocabulary and a tenth of padding: most rows of the gradient are zeros.
        dict(name="embed_grad_w1024_16384", op="embed_grad", table="bf16", dtype="bf16", rows=16384, width=1024,
             vocab=131072, padding=0.1, scale=32.0),
        # A short check in 32 bits, of odd sizes.
        dict(name="embed_grad_f32_w100_777", op="embed_grad", table="f32", dtype="f32", rows=777, width=100,
             vocab=1003, padding=0.2, scale=10.0),
        # A held-out set's score: the loss of 32,768 rows alone.
        dict(name="loss_w256_32768", op="loss", dtype="bf16", rows=32768, width=256, vocab=32768, masked=0.0),
        # The same in 32 bits at odd sizes, a third of the rows prompts that are not scored.
        dict(name="loss_f32_w100_333", op="loss", dtype="f32", rows=333, width=100, vocab=4099, masked=0.34),
        # A training step's loss and gradients at width 256, a quarter of the rows without a target.
        dict(name="loss_grad_w256_32768", op="loss_grad", dtype="bf16", rows=32768, width=256, vocab=32768, masked=0.25),
        # The largest: a wide trunk and a large vocabulary.
        dict(name="loss_grad_w1024_8192", op="loss_grad", dtype="bf16", rows=8192, width=1024, vocab=131072, masked=0.0),
        # Gradients in 32 bits at odd sizes.
        dict(name="loss_grad_f32_w200_501", op="loss_grad", dtype="f32", rows=501, width=200, vocab=5003, masked=0.1),
        # The serving loop's end: the next token of 1,024 sessions.
        dict(name="choose_w256_b1024", op="choose", dtype="bf16", rows=1024, width=256, vocab=32768),
        # One live session over a large vocabulary: latency, and the matrix read once.
        dict(name="choose_w512_b1", op="choose", dtype="bf16", rows=1, width=512, vocab=131072),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "embed_grad", "loss", "loss", "loss_grad", "loss_grad", "loss_grad", "choose",
                     "choose"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    # Widths: whole numbers of 64 as trunks have them, or any.
    width = _log(rng, 1, 32) * 64 if rng.random() < 0.6 else _log(rng, 8, 2048)
    if op.startswith("embed"):
        vocab = _log(rng, 100, min(262144, (1 << 27) // width))
        return dict(op=op, table=rng.choice([dtype, "f32"]), dtype=dtype, rows=_log(rng, 1, min(262144, (1 << 26) // width)),
                    width=width, vocab=vocab, padding=rng.choice([0.0, 0.0, 0.1, 0.5]), scale=rng.choice([1.0, width ** 0.5]))
    if op == "choose":
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 1024), width=width, vocab=_log(rng, 100, 131072))
    vocab = _log(rng, 100, 131072)
    # 32-bit products run at a sixteenth of the rate.
    most = (1 << 40) // (1 if dtype == "bf16" else 16) // (vocab * width)
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, min(32768, (1 << 30) // vocab, most)), width=width, vocab=vocab,
                masked=rng.choice([0.0, 0.0, 0.3, 0.7]))


# ---------------------------------------------------------------------------------------------
# What a program has in hand.


class _Inputs:
    """Tensors made from a seed, on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, dtype, *shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=self.gen) * scale).to(TYPES[dtype])

    def uniform32(self, lo, hi, *shape):
        return torch.rand(shape, device="cuda", generator=self.gen) * (hi - lo) + lo

    def words(self, vocab, rows):
        """Tokens as frequent as words: the v-th of the vocabulary's order in proportion to 1 / (v + 1)."""
        order = torch.randperm(vocab, device="cuda", generator=self.gen)
        share = torch.cumsum(1.0 / torch.arange(1, vocab + 1, device="cuda", dtype=torch.float64), 0)
        u = torch.rand(rows, device="cuda", generator=self.gen, dtype=torch.float64) * share[-1]
        return order[torch.searchsorted(share, u).clamp(max=vocab - 1)]

    def without(self, tokens, share):
        """The tokens with -1 in the place of some share of them."""
        tokens = tokens.clone()
        tokens[torch.randperm(len(tokens), device="cuda", generator=self.gen)[:int(len(tokens) * share)]] = -1
        return tokens


def prepare(case, seed):
    i, s = _Inputs(seed), dict(case)
    rows, width, vocab = case["rows"], case["width"], case["vocab"]
    if case["op"].startswith("embed"):
        s["E"] = i.normal(case["table"], vocab, width)
        s["tokens"] = i.without(i.words(vocab, rows), case["padding"])
        if case["op"] == "embed_grad":
            s["dy"] = i.normal(case["dtype"], rows, width, scale=0.1)
        return s
    # A head whose logits are about 1, and rows after a norm, which know their next token more or less.
    s["W"] = i.normal(case["dtype"], vocab, width, scale=width ** -0.5)
    likely = i.words(vocab, rows)
    known = i.uniform32(0.0, 12.0, rows, 1)
    s["x"] = (i.normal("f32", rows, width) + known * s["W"][likely].float()).to(TYPES[case["dtype"]])
    if case["op"] != "choose":
        s["targets"] = i.without(likely, case["masked"])
    if case["op"] == "loss_grad":  # the mean over the rows with a target, some prompts of more weight than others
        there = s["targets"] >= 0
        s["weights"] = there * i.uniform32(0.5, 1.5, rows) / max(1, rows - int(rows * case["masked"]))
    return s


# ---------------------------------------------------------------------------------------------
# One pass.


def run(state):
    return globals()["_run_" + state["op"]](state)


def _run_embed(s):
    if own:
        from uor_fbs import trunk
        return dict(y=trunk.embed(s["tokens"], s["E"], scale=s["scale"], dtype=TYPES[s["dtype"]]))
    there = s["tokens"] >= 0
    y = s["E"][s["tokens"].clamp(min=0)].float() * s["scale"]
    return dict(y=(y * there[:, None]).to(TYPES[s["dtype"]]))


def _run_embed_grad(s):
    if own:
        from uor_fbs import trunk
        return dict(dE=trunk.embed_backward(s["dy"], s["tokens"], s["E"], scale=s["scale"]))
    there = s["tokens"] >= 0
    dy = s["dy"].float() * there[:, None]
    dE = torch.zeros(s["E"].shape, device="cuda").index_add_(0, s["tokens"].clamp(min=0), dy)
    return dict(dE=(dE * s["scale"]).to(s["E"].dtype))


def _loss_plain(x, W, targets):
    """The rows' losses and logarithms of sums, which rows have a target, and their probabilities."""
    there, at = targets >= 0, targets.clamp(min=0)[:, None]
    z = x @ W.t()
    most = z.amax(1, keepdim=True)
    lse = most + torch.log(torch.exp(z - most).sum(1, keepdim=True))
    losses = (lse - z.gather(1, at))[:, 0] * there
    return losses, lse[:, 0] * there, there, at, z, lse


def _run_loss(s):
    if own:
        from uor_fbs import trunk
        losses, lse = trunk.loss(s["x"], s["W"], s["targets"])
        return dict(losses=losses, lse=lse)
    losses, lse = _loss_plain(s["x"].float(), s["W"].float(), s["targets"])[:2]
    return dict(losses=losses, lse=lse)


def _run_loss_grad(s):
    if own:
        from uor_fbs import trunk
        losses, lse = trunk.loss(s["x"], s["W"], s["targets"])
        dx, dW = trunk.loss_backward(s["weights"], s["x"], s["W"], s["targets"], lse)
        return dict(losses=losses, dx=dx, dW=dW)
    x, W = s["x"].float(), s["W"].float()
    losses, _, there, at, z, lse = _loss_plain(x, W, s["targets"])
    weights = (s["weights"] * there)[:, None]
    dz = torch.exp(z - lse) * weights
    dz.scatter_add_(1, at, -weights)
    return dict(losses=losses, dx=(dz @ W).to(s["x"].dtype), dW=(dz.t() @ x).to(s["W"].dtype))


def _run_choose(s):
    if own:
        from uor_fbs import trunk
        tokens, logprobs = trunk.choose(s["x"], s["W"])
        return dict(tokens=tokens, logprobs=logprobs)
    z = s["x"].float() @ s["W"].float().t()
    most = z.amax(1, keepdim=True)
    tokens = torch.where(z == most, torch.arange(z.shape[1], device="cuda"), z.shape[1]).amin(1)
    return dict(tokens=tokens, logprobs=-torch.log(torch.exp(z - most).sum(1)))


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without.


def _different(vocab, rows):
    """How many different tokens `rows` of _Inputs.words() are expected to have."""
    p = 1.0 / np.arange(1, vocab + 1)
    return int(-np.expm1(rows * np.log1p(-p / (p.sum() + 1e-9))).sum()) + 1


def work(case):
    op, rows, width, vocab = case["op"], case["rows"], case["width"], case["vocab"]
    size = {"bf16": 2, "f32": 4}
    if op.startswith("embed"):
        there = rows - int(rows * case["padding"])
        if op == "embed":
            read = min(_different(vocab, there), there, vocab) * width * size[case["table"]]
            return dict(bytes=8 * rows + read + rows * width * size[case["dtype"]], flops=there * width)
        return dict(bytes=8 * rows + there * width * size[case["dtype"]] + vocab * width * size[case["table"]],
                    flops=there * width)
    n = size[case["dtype"]]
    there = rows - int(rows * case.get("masked", 0.0))
    if op == "choose":
        return dict(bytes=n * width * (rows + vocab) + 12 * rows, flops=2 * rows * width * vocab)
    bytes_ = n * width * (there + vocab) + 8 * rows + 8 * rows
    if op == "loss":
        return dict(bytes=bytes_, flops=2 * there * width * vocab)
    return dict(bytes=bytes_ + n * width * (rows + vocab), flops=6 * there * width * vocab)


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits.


def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"]](s)


def _exact_embed(s):
    padded = torch.cat([s["E"].double(), s["E"].new_zeros(1, s["width"], dtype=torch.float64)])
    return dict(y=padded[s["tokens"]] * s["scale"])  # -1 is the last row, of zeros


def _exact_embed_grad(s):
    # The rows in their tokens' order, and differences of their running sums; those of padding first.
    tokens, order = torch.sort(s["tokens"], stable=True)
    ends = torch.searchsorted(tokens, torch.arange(-1, s["vocab"], device="cuda"), right=True)
    sums = torch.zeros(s["rows"] + 1, s["width"], dtype=torch.float64, device="cuda")
    torch.cumsum(s["dy"][order].double(), 0, out=sums[1:])
    return dict(dE=(sums[ends[1:]] - sums[ends[:-1]]) * s["scale"])


def _blocks(s):
    """The rows with a target, some at a time: their places, x, targets and logits."""
    W = s["W"].double()
    at = torch.nonzero(s["targets"] >= 0)[:, 0]
    for part in torch.split(at, max(1, (1 << 28) // s["vocab"])):
        x = s["x"][part].double()
        yield part, x, s["targets"][part], x @ W.t()


def _exact_loss(s):
    losses = torch.zeros(s["rows"], dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(losses)
    for part, _, target, z in _blocks(s):
        lse[part] = torch.logsumexp(z, 1)
        losses[part] = lse[part] - z[torch.arange(len(part), device="cuda"), target]
    return dict(losses=losses, lse=lse)


def _exact_loss_grad(s):
    W = s["W"].double()
    losses = torch.zeros(s["rows"], dtype=torch.float64, device="cuda")
    dx, dW = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda"), torch.zeros_like(W)
    for part, x, target, z in _blocks(s):
        row = torch.arange(len(part), device="cuda")
        log = torch.log_softmax(z, 1)
        losses[part] = -log[row, target]
        g = torch.exp(log)
        g[row, target] -= 1
        g *= s["weights"][part].double()[:, None]
        dx[part] = g @ W
        dW += g.t() @ x
    return dict(losses=losses, dx=dx, dW=dW)


def _exact_choose(s):
    log = torch.log_softmax(s["x"].double() @ s["W"].double().t(), 1)
    tokens = torch.argmax(log, 1)
    return dict(tokens=tokens, logprobs=log[torch.arange(len(tokens), device="cuda"), tokens])
