"""The oracle of a trunk's ends over its vocabulary: the embedding and the head's loss and choice, from
their definitions in 64 bits."""

import torch


def embed(tokens, table, scale):
    there = (tokens >= 0) & (tokens < table.shape[0])
    rows = table.double()[tokens.long().clamp(0, table.shape[0] - 1)] * scale
    return torch.where(there[:, None], rows, torch.zeros_like(rows))


def embed_backward(dy, tokens, vocab, scale):
    """The gradient, and the same sums over absolute values with how many rows each word has."""
    there = (tokens >= 0) & (tokens < vocab)
    at, dy = tokens[there].long(), dy.double()[there]
    grad = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=dy.device)
    return (grad.index_add(0, at, dy) * scale, grad.index_add(0, at, dy.abs()) * abs(scale),
            torch.bincount(at, minlength=vocab)[:, None])


def logits(x, weight):
    return x.double() @ weight.double().t()


def loss(x, weight, targets):
    """(losses, lse): 0 for rows whose target is outside the vocabulary."""
    there = (targets >= 0) & (targets < weight.shape[0])
    z = logits(x, weight)
    lse = torch.logsumexp(z, 1)
    losses = lse - z.gather(1, targets.long().clamp(0, weight.shape[0] - 1)[:, None])[:, 0]
    return torch.where(there, losses, torch.zeros_like(lse)), torch.where(there, lse, torch.zeros_like(lse))


def logit_gradient(x, weight, targets, dlosses, dlse):
    """(G, G without the targets' terms): the gradient at the logits."""
    there = (targets >= 0) & (targets < weight.shape[0])
    at = targets.long().clamp(0, weight.shape[0] - 1)[:, None]
    p = torch.softmax(logits(x, weight), 1)
    one = torch.zeros_like(p).scatter(1, at, 1.0)
    a = torch.zeros(len(x), dtype=torch.float64, device=x.device) if dlosses is None else dlosses.double()
    b = torch.zeros_like(a) if dlse is None else dlse.double()
    keep = there[:, None]
    g = torch.where(keep, (a + b)[:, None] * p - a[:, None] * one, torch.zeros_like(p))
    return g, g * (1 - one)


def loss_backward(dlosses, x, weight, targets, dlse=None):
    """(dx, dweight)."""
    g, _ = logit_gradient(x, weight, targets, dlosses, dlse)
    there = (targets >= 0) & (targets < weight.shape[0])
    rows = torch.where(there[:, None], x.double(), torch.zeros_like(x, dtype=torch.float64))
    return g @ weight.double(), g.t() @ rows
