"""GPU tests of a trunk's ends under autograd: what is kept for the gradients, and what has none."""

import pytest
import torch

from test_hip_trunk_ends import Make, dtype, loss_case, trunk  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("strided", [False, True])
def test_a_table_may_change_before_its_gradient(strided, dtype):  # noqa: F811
    """The lookup's gradient is none of the table's values."""
    m = Make(dtype, 3)
    table = (m(60, 24)[:, :20] if strided else m(60, 20)).requires_grad_()
    tokens, dy = m.ints(-1, 61, 90), m(90, 20)
    y = trunk.embed(tokens, table, scale=1.5)
    with torch.no_grad():
        table.mul_(2.0)
    y.backward(dy)
    assert table.grad.dtype == dtype and torch.equal(table.grad, trunk.embed_backward(dy, tokens, table.detach(), scale=1.5))


@pytest.mark.parametrize("which", ["x", "weight"])
def test_the_choice_has_no_gradient_and_says_so(which, dtype):  # noqa: F811
    x, weight, _, _ = loss_case(dtype, 20, 90, 16)
    want = trunk.choose(x, weight)
    (x if which == "x" else weight).requires_grad_()
    tokens, logprobs = trunk.choose(x, weight)
    assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1]) and not tokens.requires_grad
    with pytest.raises(trunk.TrunkError, match="choose has no gradient"):
        (logprobs.sum() + x.float().sum()).backward()
    with torch.no_grad():
        assert not trunk.choose(x, weight)[1].requires_grad
    # What the refusal names instead.
    losses, _ = trunk.loss(x, weight, tokens)
    losses.sum().backward()
    assert (x if which == "x" else weight).grad.abs().sum() > 0
