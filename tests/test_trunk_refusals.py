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
