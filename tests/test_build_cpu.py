"""What makes build() compile the binding again, beside its sources: all that its object code is made for."""
import sysconfig

import pytest
import torch

from csn_b200 import _build


@pytest.fixture
def built(monkeypatch):
    """A finished build, and the list of what further build() calls compile."""
    _build.build()
    done = []
    monkeypatch.setattr(_build, "_build_library", lambda digest, verbose: done.append("library"))
    monkeypatch.setattr(_build, "_build_binding", lambda key: done.append("binding"))
    return done


def test_nothing_changed(built):
    _build.build()
    assert built == [] and _build.last_action == "reused"


@pytest.mark.parametrize("change", ["torch", "abi", "python", "flags", "compiler", "missing"])
def test_the_binding_follows_what_it_is_built_against(built, monkeypatch, tmp_path, change):
    if change == "torch":
        monkeypatch.setattr(torch, "__version__", "99.0")
    elif change == "abi":
        monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    elif change == "python":
        real = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-399" if name == "SOABI" else real(name))
    elif change == "flags":
        monkeypatch.setattr(_build, "CXX_FLAGS", _build.CXX_FLAGS + ["-DOTHER"])
    elif change == "compiler":
        monkeypatch.setattr(_build, "_cxx_version", lambda cxx: "g++ 99")
    else:
        monkeypatch.setattr(_build, "BINDING", tmp_path / "_gated.so")
    _build.build()
    assert built == ["binding"] and _build.last_action == "built"  # the CUDA objects stay


def test_sources_make_both(built, monkeypatch):
    monkeypatch.setattr(_build, "source_hash", lambda: "0" * 16)
    _build.build()
    assert built == ["library", "binding"]


def test_key_names_no_place():
    """A tree that moves keeps its build."""
    assert _build.binding_key("x") != _build.binding_key("y")
    here = _build.binding_key("x")
    assert len(here) == 16 and here == _build.binding_key("x")
