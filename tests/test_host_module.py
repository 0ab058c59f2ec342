"""CPU: the C-ABI library and the operators do without the host-call extension (no C++ compiler, other torch headers)."""
import sys

import pytest
import torch

import orbitssm_b200 as ob
from orbitssm_b200 import _lib, build


def test_the_library_is_built_where_the_host_calls_cannot_be(monkeypatch, tmp_path):
    order = []
    monkeypatch.setattr(build, "stale", lambda: True)
    monkeypatch.setattr(build, "build_library", lambda *a: order.append("library"))
    monkeypatch.setattr(build, "HOST_OUT", str(tmp_path / "none.so"))
    monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    with pytest.warns(RuntimeWarning, match="Python host side"):
        assert build.build() == build.OUT
    assert order == ["library"]


def test_a_module_for_another_torch_is_built_again_and_not_loaded(monkeypatch, tmp_path):
    assert build.host_matches()
    monkeypatch.setattr(torch, "__version__", "1.0")
    assert not build.host_matches()
    monkeypatch.setattr(build, "_newer", lambda *a: False)
    monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    with pytest.raises(OSError):
        build.build_host()                                               # it set out to build
    monkeypatch.setattr(_lib, "_host", None)
    with pytest.warns(RuntimeWarning, match="another torch"):
        assert _lib.host().la_fwd(1, 2) is None


def test_calls_without_the_module_take_the_python_way(monkeypatch):
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setitem(sys.modules, "orbitssm_b200._orbit_host", None)
    monkeypatch.delattr(sys.modules["orbitssm_b200"], "_orbit_host", raising=False)
    with pytest.warns(RuntimeWarning, match="cannot be loaded"), pytest.raises(ValueError, match="got a CPU tensor"):
        ob.block_norm(torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(ValueError, match="got a CPU tensor"):
        ob.pack_activation(torch.zeros(2, 8))                            # (no second warning: an error under -W error)
