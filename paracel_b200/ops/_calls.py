"""Loader of ``_pcl_calls`` (built in-tree by ``paracel_b200._build``; built on first use when it is missing, or was built for another source or
another torch): the plain calls of the products by group and of the four-bit matrices, over torch's C++ interface.  Its functions return None for a
call that is not plain: the caller then goes the long way, which finds out what is wrong or different about it.  Where the module cannot be had (no
compiler, another torch) every call goes that way, and a warning says so once: the kernels are the same, a call costs the host some 6 us more."""
from __future__ import annotations

import ctypes
import importlib.util
import os
import warnings

from .. import _build
from . import _lib

_ENTRIES = ("pcl_grouped_rows", "pcl_grouped_tn", "pcl_grouped_pad", "pcl_mx4_quantize", "pcl_mx4_dequantize", "pcl_mx4_rows", "pcl_mx4_room",
            "pcl_error_string")
_mod = None


class LongWay:
    """What the module answers to calls that are not plain, for all of them."""

    @staticmethod
    def _none(*args):
        return None

    grouped_rows = grouped_tn = quantize = dequantize = mx4_rows = _none


def calls():
    global _mod
    if _mod is None:
        lib = _lib.load()                                # without the kernels there is no other way: this raises
        try:
            _mod = _module(lib)
        except Exception as e:
            warnings.warn(f"products by group and four-bit matrices are called through Python, some 6 us a call slower: {e}", RuntimeWarning, stacklevel=3)
            _mod = LongWay
    return _mod


def _module(lib):
    path = _build.calls_path()
    if not _build.calls_current():
        if os.environ.get("PCL_NO_AUTOBUILD", "0") == "1":
            raise _lib.KernelLibraryMissing(f"{path} is missing or was built for another torch; run python -m paracel_b200._build")
        _build.build_calls()
    spec = importlib.util.spec_from_file_location("_pcl_calls", str(path))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _ENTRIES))
    return mod
