"""GPU tests of the float trunk's operators (uor_fbs.trunk): values near a rounding's border.

A bf16 output is half a step off at most wherever it is computed from; what shows how it was computed is
which way it rounds. The outputs here are single products whose exact value is 2^-19 of itself away from
the middle between two bf16 numbers. In 32 bits a product is off by 2^-24 of itself, a step (softplus)
by 2^-21 at most, and a weight goes through at most four such products: together under 2^-20, so that the
output has to be the exact value's rounding. Of an operand in two bf16 parts, 2^-18 is missing.
"""

import pytest
import torch

import trunk_cases as oracle

pytestmark = pytest.mark.gpu
trunk = pytest.importorskip("uor_fbs.trunk")
BF16 = torch.bfloat16


def borders(*shape, seed=1):
    """Values in 64 bits, each 2^-19 of itself from the middle between two bf16 numbers."""
    g = torch.Generator().manual_seed(seed)
    middle = 1 + torch.randint(0, 128, shape, generator=g).double() / 128 + 1 / 256
    sign = torch.randint(0, 2, shape, generator=g).double() * 2 - 1
    scale = 2.0 ** torch.randint(-3, 4, shape, generator=g).double()
    return middle * (1 + sign * 2.0 ** -19) * scale


def parts(v):
    """v as three bf16 numbers whose sum is v to 2^-25 of it, along a new last axis."""
    out = []
    for _ in range(3):
        out.append(v.to(BF16))
        v = v - out[-1].double()
    return torch.stack(out, -1)


def gpu(*tensors):
    return [t.cuda() for t in tensors]


def test_states_reach_y_in_32_bits():
    """Steps of nothing: the state stands still, and a C of one place reads one value of it."""
    rows, heads, dim, state = 70, 2, 64, 64
    h = borders(1, heads, dim, state).float()
    C = torch.zeros(rows, 1, state, dtype=BF16)
    C[torch.arange(rows), 0, torch.arange(rows) % state] = 1
    x, dt, A, B, Cd, hd = gpu(torch.zeros(rows, heads, dim, dtype=BF16), torch.full((rows, heads), -200.0, dtype=BF16), torch.full((heads,), -1.0),
                              torch.zeros(rows, 1, state, dtype=BF16), C, h)
    y, final = trunk.scan(x, dt, A, B, Cd, initial=hd)
    assert torch.equal(final, hd)
    want = h[0].to(BF16)  # (head, value, place)
    for t in range(rows):
        assert torch.equal(y[t].cpu(), want[:, :, t % state]), t


def test_weights_reach_y_in_32_bits():
    """Weights of rows: the skip, and C_t . B_s with a step of one row, in every tile before and at its own."""
    rows, dim, state = 64, 64, 16
    step = torch.tensor([0.75]).to(BF16)
    wide = oracle.softplus(step.double())
    # Row s alone has x, at value s: y[t, s] = (C_t . B_s) D x, of a C_t whose three places sum to what is wanted.
    x = torch.eye(rows, dim).to(BF16)[:, None]
    goal = borders(rows)
    C = torch.zeros(rows, 1, state, dtype=BF16)
    C[:, 0, :3] = parts(goal / wide)
    B = torch.zeros(rows, 1, state, dtype=BF16)
    B[:, 0, :3] = 1
    xd, dt, A, Bd, Cd = gpu(x, step.expand(rows, 1).contiguous(), torch.zeros(1), B, C)
    y, _ = trunk.scan(xd, dt, A, Bd, Cd)
    want = torch.tril(goal.to(BF16)[:, None].expand(rows, dim))
    assert torch.equal(y[:, 0].cpu(), want)
    D = borders(40, seed=2).float()
    ones = torch.ones(9, 40, 33, dtype=BF16)
    y, _ = trunk.scan(*gpu(ones, torch.zeros(9, 40, dtype=BF16), -torch.ones(40), torch.zeros(9, 2, 16, dtype=BF16), torch.zeros(9, 2, 16, dtype=BF16)),
                      D=D.cuda())
    assert torch.equal(y.cpu(), D.to(BF16)[None, :, None].expand(9, 40, 33))


def gradient(dy, x, dt, B, C, **other):
    heads = x.shape[1]
    other = {k: v.cuda() for k, v in other.items()}
    return trunk.scan_backward(*gpu(dy, x, dt, torch.zeros(heads), B, C), **other)


def test_weights_reach_the_gradients_in_32_bits():
    """dx, dB and dC of single weights, with decays of one."""
    n = 64
    step = torch.full((n, 1), 0.75, dtype=BF16)
    wide = oracle.softplus(step.double())[0, 0]
    one_hot, three = torch.eye(n).to(BF16)[:, None], torch.zeros(n, 1, n, dtype=BF16)
    ones = torch.zeros(n, 1, n, dtype=BF16)
    ones[:, 0, :3] = 1
    goal = borders(n, seed=3)
    three[:, 0, :3] = parts(goal / wide)
    none = torch.zeros(n, 1, n, dtype=BF16)
    want = goal.to(BF16)
    # dy_t is one at value t: dx[s, t] = D C_t . B_s for s <= t.
    got = gradient(one_hot, none, step, ones, three)
    assert torch.equal(got.dx[:, 0].cpu(), torch.triu(want[None].expand(n, n)))
    # W_ts = dy_t . x_s; C_t is one at place t: dB[s, t] = D W_ts for s <= t.
    got = gradient(three, ones, step, none, one_hot)
    assert torch.equal(got.dB[:, 0].cpu(), torch.triu(want[None].expand(n, n)))
    # B_s is one at place s: dC[t, s] = W_ts D for s <= t.
    got = gradient(three, ones, step, one_hot, none)
    assert torch.equal(got.dC[:, 0].cpu(), torch.tril(want[:, None].expand(n, n)))


def test_states_reach_the_gradients_in_32_bits():
    """dB and dx of a gradient at the final state, dC of an initial one."""
    n = 64
    step = torch.full((n, 1), 0.75, dtype=BF16)
    wide = oracle.softplus(step.double())[0, 0]
    one_hot, none = torch.eye(n).to(BF16)[:, None], torch.zeros(n, 1, n, dtype=BF16)
    goal = borders(n, n, seed=4)
    state = (goal / wide).float()[None, None]
    got = gradient(none, one_hot, step, one_hot, none, dfinal=state)
    assert torch.equal(got.dB[:, 0].cpu(), goal.to(BF16))      # x_s is one at value s: dB[s] = D g[s, :]
    assert torch.equal(got.dx[:, 0].cpu(), goal.to(BF16).t())  # B_s is one at place s: dx[s] = D g[:, s]
    got = gradient(one_hot, none, step, none, none, initial=goal.float()[None, None])
    assert torch.equal(got.dC[:, 0].cpu(), goal.to(BF16))      # dy_t is one at value t: dC[t] = h[t, :]


# ---------------------------------------------------------------------------------------------
# The activation's tails. In 32 bits e^-v is off by at most 4 x 2^-24 of itself (the exponential's and its
# argument's last bits, and their product), the sum and the reciprocal by 2 x 2^-24, and each product
# after by 2^-24: under 16 x 2^-24 of the value itself, however small it is.
SIGMOID = 16 * 2.0 ** -24


def tails():
    return torch.cat([torch.linspace(-86, 86, 4001), torch.linspace(-2, 2, 95)]).float()


def relative(got, want, unit):
    off = (got.cpu().double() - want).abs()
    bad = ~(off <= unit * want.abs())
    assert not bad.any(), (int(bad.sum()), float((off / want.abs())[bad].max() * 2 ** 24))


def test_silu_keeps_its_bits_for_negative_values():
    """One tap of one: y = v sigmoid(v), as the convolution computes it and its step."""
    v = tails()
    want = v.double() / (1 + torch.exp(-v.double()))
    w = torch.ones(v.numel(), 1)
    y, _ = trunk.conv(*gpu(v[None], w))
    relative(y[0], want, SIGMOID)
    y = trunk.conv_step(*gpu(v[None], w), torch.zeros(1, 0, v.numel()).cuda())
    relative(y[0], want, SIGMOID)


def test_silu_slopes_keep_their_bits_for_negative_values():
    """sigmoid(v) (1 + v sigmoid(-v)), but where its two terms cancel: there, relative to them."""
    v = tails()
    wide = v.double()
    s = 1 / (1 + torch.exp(-wide))
    want = s * (1 + wide * (1 - s))
    size = s * (1 + wide.abs() * (1 - s))
    got = trunk.conv_backward(*gpu(torch.ones(1, v.numel()), v[None], torch.ones(v.numel(), 1)))
    off = (got.dx[0].cpu().double() - want).abs()
    assert not (off > SIGMOID * size).any(), float((off / size).max() * 2 ** 24)


def test_gates_keep_their_bits_for_negative_values():
    """Rows of one value: with a large eps the norm is a factor that is known."""
    v = tails()
    rows, one = v[:, None].contiguous(), torch.ones(v.numel(), 1)
    wide = v.double()
    gated = wide / (1 + torch.exp(-wide))
    want = gated / torch.sqrt(gated * gated + 1e12)
    r, _ = trunk.norms(None, *gpu(one), gate=rows.cuda(), eps=1e12)
    whole = want.abs() >= 2.0 ** -126  # numbers below have fewer bits, whoever computes them
    assert whole.sum() > 3500
    relative(r[:, 0].cpu()[whole], want[whole], 2 * SIGMOID)


def test_step_slopes_keep_their_bits_for_negative_steps():
    """ddt = (x . g B) sigmoid(dt) with a decay of one, for steps down to e^-80."""
    v = tails()
    n = v.numel()
    one = torch.ones(n, 1, 1)
    got = trunk.scan_backward(*gpu(torch.zeros(n, 1, 1), one, v[:, None].contiguous(), torch.zeros(1), one, torch.zeros(n, 1, 1)),
                              dfinal=torch.ones(1, 1, 1, 1).cuda())
    relative(got.ddt[:, 0], 1 / (1 + torch.exp(-v.double())), 2 * SIGMOID)


def test_silu_of_infinities():
    v = torch.tensor([[float("inf"), float("-inf"), float("nan"), 200.0, -200.0, 0.0]])
    y, _ = trunk.conv(*gpu(v, torch.ones(6, 1)))
    y = y[0].tolist()
    assert y[0] == float("inf") and y[2] != y[2] and y[3] == 200.0 and abs(y[4]) < 1e-34 and y[5] == 0.0


def test_a_step_that_is_no_number_has_no_gradient():
    one = torch.ones(1, 1, 1)
    for dtype in (torch.float32, BF16):
        got = trunk.scan_backward(*gpu(one.to(dtype), one.to(dtype), torch.full((1, 1), float("nan"), dtype=dtype), torch.zeros(1), one.to(dtype),
                                       one.to(dtype)))
        assert got.ddt.isnan().all() and got.dx.isnan().all() and not got.dC.isfinite().any()
