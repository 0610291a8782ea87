"""The module of plain calls (`ops/_calls.py`) is bound to torch's C++ interface: one that was built for another torch is never loaded, and where it
cannot be built the calls go the way through Python."""
import types
import warnings

import pytest

from paracel_b200 import _build
from paracel_b200.ops import _calls, _lib

NAMES = ("grouped_rows", "grouped_tn", "quantize", "dequantize", "mx4_rows")


@pytest.fixture
def place(monkeypatch, tmp_path):
    """An empty folder of built files, a kernel library that nothing calls, no module loaded; the list gets what is built."""
    built = []
    monkeypatch.setattr(_build, "LIB", tmp_path)
    monkeypatch.setattr(_calls, "_mod", None)
    monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace())
    monkeypatch.delenv("PCL_NO_AUTOBUILD", raising=False)

    def build_calls(*a, **k):
        built.append(_build.calls_path())
        raise RuntimeError("no compiler here")

    monkeypatch.setattr(_build, "build_calls", build_calls)
    return built


def _all_go_the_long_way(words):
    with pytest.warns(RuntimeWarning, match=words):
        mod = _calls.calls()
    assert all(getattr(mod, name)(1, 2, 3) is None for name in NAMES)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert _calls.calls() is mod                     # said once


def test_a_missing_module_that_cannot_be_built(place):
    _all_go_the_long_way("no compiler here")
    assert place == [_build.calls_path()]


@pytest.mark.parametrize("stamp", [None, "of another torch"])
def test_a_stale_module_is_not_loaded(place, stamp):
    _build.calls_path().write_bytes(b"built for another torch")
    if stamp is not None:
        (_build.LIB / "calls.stamp").write_text(stamp)
    assert not _build.calls_current()
    _all_go_the_long_way("no compiler here")
    assert place == [_build.calls_path()]


def test_nothing_is_built_where_that_is_switched_off(place, monkeypatch):
    monkeypatch.setenv("PCL_NO_AUTOBUILD", "1")
    _all_go_the_long_way("_build")
    assert place == []


def test_a_module_that_does_not_load(place):
    _build.calls_path().write_bytes(b"not a shared object")
    (_build.LIB / "calls.stamp").write_text(_build._calls_stamp())
    assert _build.calls_current()
    _all_go_the_long_way("")
    assert place == []


def test_the_stamp_follows_torch_and_the_source_but_not_the_place(monkeypatch, tmp_path):
    import torch
    here = _build._calls_stamp()
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    other = _build._calls_stamp()
    assert other != here
    monkeypatch.undo()
    (tmp_path / "calls").mkdir()
    copy = tmp_path / "calls" / "calls.cpp"
    copy.write_bytes((_build.CSRC / "calls" / "calls.cpp").read_bytes())
    monkeypatch.setattr(_build, "CSRC", tmp_path)
    assert _build._calls_stamp() == here
    copy.write_text(copy.read_text() + "//")
    assert _build._calls_stamp() != here


def test_without_the_kernels_there_is_no_long_way(monkeypatch):
    def load():
        raise _lib.KernelLibraryMissing("no kernels")

    monkeypatch.setattr(_calls, "_mod", None)
    monkeypatch.setattr(_lib, "load", load)
    with pytest.raises(_lib.KernelLibraryMissing):
        _calls.calls()
