"""GPU tests of the small float trunk without logits (Config.keep_logits false): its gradients against 64 bits and its replies.

The bound on a logit's or a gradient's error is that of the trunk with logits: at most 2 layers x 8 sums each way, of
at most 128 terms, off by 2^-24 a term of their absolute sum, 32 x 128 x 12 x 2^-24 = 3e-3 of the whole's norm.
"""

import pytest
import torch
import torch.nn.functional as F

from test_hip_float_trunk import close, config, ft, plain, ragged

pytestmark = pytest.mark.gpu


def test_gradients_against_64_bits():
    cfg = config(keep_logits=False)
    p = ft.make_params(cfg, 3)
    tokens, offsets = ragged([5, 0, 70, 1], cfg.vocab)
    targets = torch.randint(-1, cfg.vocab, (76,), generator=torch.Generator().manual_seed(1)).cuda()
    loss, grads = ft.gradients(cfg, p, tokens, targets, offsets)
    wide = {k: v.detach().cpu().double().requires_grad_() for k, v in p.items()}
    want = F.cross_entropy(plain(cfg, wide, tokens, offsets), targets.cpu(), ignore_index=-1)
    want.backward()
    close(loss.reshape(1), want.reshape(1), "loss")
    assert set(grads) == set(p)
    for k, v in wide.items():
        close(grads[k], v.grad, k)


def test_a_target_outside_the_vocabulary_is_none():
    cfg = config(keep_logits=False)
    p = ft.make_params(cfg, 3)
    tokens, offsets = ragged([5, 20], cfg.vocab)
    targets = tokens.roll(-1)
    targets[[3, 11]] = -1
    want = ft.gradients(cfg, p, tokens, targets, offsets)
    targets[11] = cfg.vocab
    got = ft.gradients(cfg, p, tokens, targets, offsets)
    assert torch.equal(got[0], want[0]) and all(torch.equal(got[1][k], v) for k, v in want[1].items())


def test_replies_are_those_of_the_logits():
    cfg = config()
    p = ft.make_params(cfg, 4)
    tokens, offsets = ragged([9, 30, 2], cfg.vocab)
    said = []
    for keep in (True, False):
        one = cfg._replace(keep_logits=keep)
        said.append(ft.reply(one, p, tokens, offsets, 6, ft.make_state(one, 7), torch.tensor([6, 0, 3], dtype=torch.int32).cuda()))
    assert torch.equal(*said)


def test_the_step_of_a_bf16_trunk_runs():
    cfg = ft.Config(vocab=300, width=64, layers=2, keep_logits=False)
    p = ft.make_params(cfg)
    losses = ft.train(cfg, p, 3, count=8, length=6)
    assert all(0 < v < 100 for v in losses)
    assert all(torch.isfinite(t).all() for t in p.values())
