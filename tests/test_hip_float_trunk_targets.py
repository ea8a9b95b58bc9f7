"""GPU tests of the small float trunk: targets that are none, tokens and tables that a lookup does not take as they are."""

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


def test_tokens_and_tables_that_a_lookup_does_not_take_as_they_are():
    """Tokens on the CPU, a table of another type, a row and a word more than a lookup takes."""
    cfg = config(vocab=(1 << 23) + 1, width=8, layers=1, heads=1, groups=1, dim=4, state=4)
    p = ft.make_params(cfg, 3)
    tokens, offsets = torch.tensor([5, 1 << 23, 0, 77]), torch.tensor([0, 4], dtype=torch.int32).cuda()
    want = ft.prompts(cfg, {**p, "embed": p["embed"][tokens.cuda()]}, torch.arange(4).cuda(), offsets)
    assert torch.equal(ft.prompts(cfg, p, tokens, offsets), want)
    half = {**p, "embed": p["embed"][:100].half()}
    assert torch.equal(ft.prompts(cfg, half, tokens % 100, offsets), ft.prompts(cfg, {**half, "embed": half["embed"].float()}, tokens % 100, offsets))
    del want
    few = config(vocab=8, width=8, layers=1, heads=1, groups=1, dim=4, state=4)
    p = ft.make_params(few, 3)
    tokens, offsets = torch.arange((1 << 24) + 1, device="cuda") % 5, torch.tensor([0, 3, (1 << 24) - 2, (1 << 24) + 1], dtype=torch.int32).cuda()
    got = ft._prompt_rows(few, p, tokens, offsets)[-3:]
    assert torch.equal(got, ft._prompt_rows(few, p, tokens[-3:], torch.tensor([0, 3], dtype=torch.int32).cuda()))
    torch.cuda.empty_cache()
