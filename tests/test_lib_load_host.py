"""A library that was built before an entry point was added is refused with a word about it, not with an AttributeError (no GPU needed)."""
import ctypes

import pytest

import avsi_amd  # noqa: F401
from avsi_amd import _lib


def test_an_older_library_is_named(monkeypatch):
    _lib.lib()
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setitem(_lib.PROTOTYPES, "avsi_added_after_the_build", (ctypes.c_int, []))
    with pytest.raises(_lib.AvsiError, match="no avsi_added_after_the_build.*rebuild"):
        _lib.lib()
