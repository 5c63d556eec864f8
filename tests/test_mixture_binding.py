"""The mixture operators' binding is there: without it, these tests fail, where a test that asks with importorskip is skipped."""
import subprocess
import sys

import pytest


@pytest.mark.parametrize("where", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
def test_the_binding_loads(where):
    from provenloop_amd import mixture

    assert mixture._ext.__file__.endswith("_mixture_torch.so")


def test_build_loads_it(monkeypatch):
    """build() ends with an error if the binding that it has built cannot be imported."""
    import __graft_entry__

    monkeypatch.setattr(subprocess, "run", lambda *a, **k: None)
    __graft_entry__.build()
    monkeypatch.setitem(sys.modules, "provenloop_amd.mixture", None)
    with pytest.raises(ImportError):
        __graft_entry__.build()


def test_a_missing_binding_says_how_to_build_it(monkeypatch):
    import provenloop_amd

    monkeypatch.delattr(provenloop_amd, "_mixture_torch", raising=False)
    monkeypatch.delitem(sys.modules, "provenloop_amd.mixture", raising=False)
    monkeypatch.setitem(sys.modules, "provenloop_amd._mixture_torch", None)
    with pytest.raises(ImportError, match="make -C provenloop_amd/csrc mixture"):
        import provenloop_amd.mixture  # noqa: F401
