"""Loader of ``_pcl_calls`` (built in-tree by ``paracel_b200._build``; built on first use when it is missing): the plain calls of the
products by group and of the four-bit matrices, over torch's C++ interface.  Its functions return None for a call that is not plain: the
caller then goes the long way, which finds out what is wrong or different about it."""
from __future__ import annotations

import ctypes
import importlib.util
import os

from .. import _build
from . import _lib

_ENTRIES = ("pcl_grouped_rows", "pcl_grouped_tn", "pcl_grouped_pad", "pcl_mx4_quantize", "pcl_mx4_dequantize", "pcl_mx4_rows", "pcl_mx4_room",
            "pcl_error_string")
_mod = None


def calls():
    global _mod
    if _mod is None:
        lib = _lib.load()
        path = _build.calls_path()
        if not path.exists():
            if os.environ.get("PCL_NO_AUTOBUILD", "0") == "1":
                raise _lib.KernelLibraryMissing(f"{path} is missing; run python -m paracel_b200._build")
            _build.build_calls()
        spec = importlib.util.spec_from_file_location("_pcl_calls", str(path))
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _ENTRIES))
        _mod = mod
    return _mod
