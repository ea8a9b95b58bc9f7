"""GPU tests of a trunk's ends at values where their precision shows."""

import pytest
import torch

import ends_cases as oracle
from test_hip_trunk_ends import Make, dtype, trunk  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,width", [(20, 300, 32), (20, 30000, 64), (100, 300, 32), (400, 3000, 64), (3000, 3000, 64)])
def test_the_loss_of_a_sure_row_does_not_grow_with_its_logit(rows, vocab, width, dtype):  # noqa: F811
    """Rows of logits up to some 2,000 whose target's share is 1 but for 2^-30. What is left is that share's own error: an
    exponential's, good to 2^-22 of itself, of an exponent near 0 that is a difference taken exactly, and the logit's sums do not
    come in, as the loss is a difference of the same one. So 2^-21 bounds it, at any logit."""
    m = Make(dtype, rows + vocab)
    weight, targets = m(vocab, width), torch.arange(rows).cuda() % vocab
    x = (weight[targets].float() * torch.linspace(1, 30, rows).cuda()[:, None]).to(dtype)
    sure = oracle.loss(x, weight, targets)[0] < 2.0 ** -30
    assert sure.sum() > rows // 4
    assert trunk.loss(x, weight, targets)[0][sure].abs().max() <= 2.0 ** -21
    tokens, logprobs = trunk.choose(x, weight)
    assert torch.equal(tokens[sure], targets[sure]) and logprobs[sure].abs().max() <= 2.0 ** -21
