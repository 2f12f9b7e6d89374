"""Host logic around the scan-wise operators: a library of other sources, limits of a launch, checkpoints, known batches (no GPU)."""
import pytest
import torch


def test_a_library_of_other_sources_is_named_as_such(monkeypatch):
    """A library without an entry point that this package calls (built before it existed) is a version mismatch, not an AttributeError."""
    from lidiff_amd import _lib
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setitem(_lib.SIGNATURES, "lidiff_of_a_later_version", (_lib._i32, []))
    with pytest.raises(RuntimeError, match="version mismatch.*lidiff_of_a_later_version"):
        _lib.load()
    monkeypatch.undo()
    assert _lib.load().lidiff_abi_version() == _lib.ABI_VERSION
