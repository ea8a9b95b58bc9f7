"""GPU tests of uor_fbs.trunk under autograd: gradients are those of the *_backward calls, bit for bit,
steps have none and say so, and what they change in place is seen."""

import pytest
import torch

from test_hip_trunk import Make, conv_case, dtype, scan_case, trunk  # noqa: F401

pytestmark = pytest.mark.gpu


def leaves(x):
    return {k: v.detach().clone().requires_grad_() if v is not None and v.is_floating_point() else v for k, v in x.items()}


def same(got, want):
    assert (got is None) == (want is None)
    assert got is None or torch.equal(got, want)


@pytest.mark.parametrize("used", ["y", "final", "both"])
def test_scan(used, dtype):
    x, m = scan_case(dtype, [70, 0, 30], 4, 2, 24, 16, initial=True)
    dy, df = m(*x["x"].shape), m.f32(3, 4, 24, 16)
    if used == "final":
        dy.zero_()
    w = leaves(x)
    y, final = trunk.scan(**w)
    want = trunk.scan(**x)
    assert torch.equal(y, want[0]) and torch.equal(final, want[1]) and y.requires_grad and final.requires_grad
    outs = {"y": ([y], [dy]), "final": ([final], [df]), "both": ([y, final], [dy, df])}[used]
    torch.autograd.backward(*outs)
    got = trunk.scan_backward(dy, **x, dfinal=None if used == "y" else df)
    for name in ("x", "dt", "A", "B", "C", "D", "dt_bias", "initial"):
        same(w[name].grad, getattr(got, "d" + name))


def test_scan_within_a_larger_expression(dtype):
    """Views, absent parameters, a loss that hands back one value for all, and inputs of no gradient."""
    x, m = scan_case(dtype, [40, 9], 2, 1, 16, 16)
    rows = torch.cat([x["x"].flatten(1), x["B"].flatten(1)], 1).requires_grad_()
    A = x["A"].log().nan_to_num(0.0).requires_grad_()
    y, _ = trunk.scan(rows[:, :32].unflatten(1, (2, 16)), x["dt"], -A.exp(), rows[:, 32:].unflatten(1, (1, 16)), x["C"], offsets=x["offsets"])
    y.float().sum().backward()
    got = trunk.scan_backward(torch.ones_like(y), x["x"], x["dt"], -A.detach().exp(), x["B"], x["C"], offsets=x["offsets"])
    same(rows.grad, torch.cat([got.dx.flatten(1), got.dB.flatten(1)], 1))
    same(A.grad, got.dA * -A.detach().exp())


@pytest.mark.parametrize("silu", [True, False])
def test_conv(silu, dtype):
    x, m = conv_case(dtype, [30, 0, 2, 9], 12, 4, True)
    w = leaves(x)
    y, final = trunk.conv(**w, silu=silu)
    dy, df = m(*y.shape), m(*final.shape)
    torch.autograd.backward([y, final], [dy, df])
    got = trunk.conv_backward(dy, **x, dfinal=df, silu=silu)
    for name in ("x", "weight", "bias", "initial"):
        same(w[name].grad, getattr(got, "d" + name))


@pytest.mark.parametrize("absent", [(), ("gate",), ("residual",), ("out", "gate", "post", "scale"), ("pre",)], ids=str)
def test_norms(absent, dtype):
    m = Make(dtype, 4)
    x = dict(residual=m(9, 40), out=m(9, 40), gate=m(9, 40), post=m.f32(40), scale=m.f32(40), pre=m.f32(40))
    x = {k: None if k in absent else v for k, v in x.items()}
    w = leaves(x)
    r, n = trunk.norms(**w)
    dr, dn = m(9, 40), None if n is None else m(9, 40)
    if "out" in absent:
        assert r is w["residual"]
        n.backward(dn)
        got = trunk.norms_backward(None, dn, **x)
    else:
        torch.autograd.backward([r] + [n] * (n is not None), [dr] + [dn] * (n is not None))
        got = trunk.norms_backward(dr, dn, **x)
    for name in x:
        same(None if w[name] is None else w[name].grad, getattr(got, "d" + name))


def test_without_gradients_there_is_no_history(dtype):
    x, _ = scan_case(dtype, [20], 2, 1, 16, 16)
    w = leaves(x)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            y, final = trunk.scan(**w)
            assert not y.requires_grad and not final.requires_grad
    assert trunk.scan(**x)[0].grad_fn is None


def test_second_derivatives_raise(dtype):
    x, _ = scan_case(dtype, [20], 2, 1, 16, 16)
    w = leaves(x)
    y, _ = trunk.scan(**w)
    g, = torch.autograd.grad(y.float().square().sum(), w["x"], create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_steps_have_no_gradient_and_say_so(dtype):
    x, m = scan_case(dtype, [3], 2, 1, 16, 16)
    one = {k: x[k] for k in ("x", "dt", "A", "B", "C")}
    states = m.f32(3, 2, 16, 16)
    other = states.clone()
    want = trunk.scan_step(**one, states=states)
    y = trunk.scan_step(**leaves(one), states=other)
    assert torch.equal(y, want) and torch.equal(states, other)
    with pytest.raises(trunk.TrunkError, match="scan_step has no gradient"):
        y.float().sum().backward()
    c, m = conv_case(dtype, [3], 8, 4, False)
    held = m(3, 3, 8)
    y = trunk.conv_step(c["x"], c["weight"].clone().requires_grad_(), held)
    with pytest.raises(trunk.TrunkError, match="conv_step has no gradient"):
        y.float().sum().backward()
    with torch.inference_mode():
        inside = torch.zeros(3, 2, 16, 16, device="cuda")
        trunk.scan_step(**one, states=inside)
        assert inside.any()


def test_states_that_a_step_changes_are_seen_to_change(dtype):
    """A state that a gradient still needs is not the same after a step over it."""
    x, m = scan_case(dtype, [3], 2, 1, 16, 16)
    states = m.f32(1, 2, 16, 16)
    w = leaves({k: x[k] for k in ("x", "dt", "A", "B", "C")})
    y, _ = trunk.scan(**w, initial=states)
    trunk.scan_step(**{k: x[k][:1] for k in ("x", "dt", "B", "C")}, A=x["A"], states=states)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
