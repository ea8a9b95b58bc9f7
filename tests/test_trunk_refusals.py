"""What uor_fbs.trunk refuses beside wrong arguments, on the CPU."""

import pytest
import torch

trunk = pytest.importorskip("uor_fbs.trunk")


class OlderLibrary:
    """A library built before some of the calls were there."""

    def __init__(self, path):
        pass

    def __getattr__(self, name):
        if name not in ("uor_trunk_abi_version", "uor_trunk_last_error", "uor_trunk_sizeof_scan"):
            raise AttributeError(name)
        call = {"uor_trunk_abi_version": lambda: trunk.ABI_VERSION, "uor_trunk_sizeof_scan": lambda: trunk.C.sizeof(trunk.CScan)}.get(name, lambda: b"")
        return type("Call", (), {"__call__": staticmethod(call)})()


def test_a_library_without_the_calls_is_of_another_version(monkeypatch):
    monkeypatch.setattr(trunk, "_lib", None)
    monkeypatch.setattr(trunk, "LIB_PATH", __file__)
    monkeypatch.setattr(trunk.C, "CDLL", OlderLibrary)
    with pytest.raises(trunk.TrunkError, match="is of another version: build it again"):
        trunk.lib()


def test_forward_mode_derivatives_are_refused():
    """They are not computed: a tangent would be lost without a word."""
    f32, ints = torch.zeros, torch.zeros(4, dtype=torch.int64)
    with torch.autograd.forward_ad.dual_level():
        one = torch.autograd.forward_ad.make_dual(f32(4, 8), torch.ones(4, 8))
        calls = [lambda: trunk.embed(ints, one), lambda: trunk.loss(one, f32(9, 8), ints), lambda: trunk.loss(f32(4, 8), one, ints),
                 lambda: trunk.choose(one, f32(9, 8)), lambda: trunk.embed_backward(one, ints, f32(9, 8)), lambda: trunk.norms(one, pre=f32(8)),
                 lambda: trunk.conv(one, f32(8, 2)), lambda: trunk.conv_step(one, f32(8, 2), f32(4, 1, 8)),
                 lambda: trunk.scan(one[..., None], f32(4, 8), f32(8), f32(4, 1, 2), f32(4, 1, 2)),
                 lambda: trunk.embed(ints, one[:, 2:6])]
        for call in calls:
            with pytest.raises(trunk.TrunkError, match="forward-mode"):
                call()
        with pytest.raises(trunk.TrunkError, match="on cpu"):  # no tangent among them
            trunk.embed(ints, f32(4, 8))
    with pytest.raises(trunk.TrunkError, match="on cpu"):
        trunk.embed(ints, f32(4, 8))


def test_forward_mode_derivatives_beside_gradients_are_refused():
    weight = torch.zeros(9, 8, requires_grad=True)
    with torch.autograd.forward_ad.dual_level():
        one = torch.autograd.forward_ad.make_dual(torch.zeros(4, 8), torch.ones(4, 8))
        with pytest.raises(trunk.TrunkError, match="forward-mode"):
            trunk.loss(one, weight, torch.zeros(4, dtype=torch.int64))
        with pytest.raises(trunk.TrunkError, match="forward-mode"):
            trunk.norms(one, pre=torch.zeros(8, requires_grad=True))
