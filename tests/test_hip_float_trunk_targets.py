"""GPU tests of the small float trunk's targets that are none."""

import pytest
import torch

from test_hip_float_trunk import config, ft, ragged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep", [True, False], ids=["logits", "no logits"])
def test_a_target_outside_the_vocabulary_is_none(keep):
    cfg = config(keep_logits=keep)
    p = ft.make_params(cfg, 3)
    tokens, offsets = ragged([5, 20], cfg.vocab)
    targets = tokens.roll(-1)
    targets[[3, 11, 24]] = -1
    want = ft.gradients(cfg, p, tokens, targets, offsets)
    targets[3], targets[11], targets[24] = cfg.vocab, cfg.vocab + 1, 1 << 40
    got = ft.gradients(cfg, p, tokens, targets, offsets)
    assert torch.equal(got[0], want[0]) and all(torch.equal(got[1][k], v) for k, v in want[1].items())
