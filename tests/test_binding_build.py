"""The Python binding belongs to the torch and the Python that it was built with."""
import os

import pytest
import torch

from heterocache_b200 import _lib
from heterocache_b200 import build as b


@pytest.fixture(scope="module", autouse=True)
def _built():
    b.build()


def test_a_binding_of_this_torch_is_kept():
    assert not b._binding_stale()
    before = os.path.getmtime(b.BINDING_OUT)
    b.build()
    assert os.path.getmtime(b.BINDING_OUT) == before


@pytest.mark.parametrize("what", ["__version__", "git_version", "abi", "python"])
def test_another_torch_makes_it_stale(monkeypatch, what):
    """Whatever the files' times: another torch may well be older than the binding."""
    if what == "__version__":
        monkeypatch.setattr(torch, "__version__", "2.0.0")
    elif what == "git_version":
        monkeypatch.setattr(torch.version, "git_version", "0" * 40)
    elif what == "abi":
        monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: False)
    else:
        monkeypatch.setattr(b.sys.implementation, "cache_tag", "cpython-300")
    assert b._binding_stale()


def test_it_is_not_loaded_into_another_torch(monkeypatch):
    monkeypatch.setattr(_lib, "_PAGED", None)
    monkeypatch.setattr(torch, "__version__", "2.0.0")
    with pytest.raises(RuntimeError, match="built for another torch"):
        _lib.paged()
    monkeypatch.undo()
    assert _lib.paged() is not None
