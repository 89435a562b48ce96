"""
ctypes binding of ``librtn_model_ops.so`` (C ABI declared in ``include/rtn_model_ops.h``) and the torch side of its
calls (``_rtn_model.so``).  As for the other libraries there is no fallback: what has not been built raises.
"""

from __future__ import annotations

import ctypes
import os
import threading
from typing import Optional

from . import build as _build
from .lib import NativeLibraryMismatch, NativeLibraryMissing

# The ABI version the argument lists below were written for (rtn_model_ops_abi_version()).
EXPECTED_ABI = 1

# every symbol include/rtn_model_ops.h declares
SYMBOLS = (
    "rtn_model_ops_abi_version",
    "rtn_model_ops_last_error",
    "rtn_delta_rule_fwd_workspace_bytes",
    "rtn_delta_rule_saved_bytes",
    "rtn_delta_rule_fwd",
    "rtn_delta_rule_bwd_workspace_bytes",
    "rtn_delta_rule_bwd",
    "rtn_embedding_fwd",
    "rtn_embedding_bwd_workspace_bytes",
    "rtn_embedding_bwd",
    "rtn_beam_select_workspace_bytes",
    "rtn_beam_select",
    "rtn_reorder_rows",
)

_lock = threading.RLock()
_lib: Optional[ctypes.CDLL] = None
_native_module = None


def load() -> ctypes.CDLL:
    """Load the built library (once per process). Never builds, never falls back."""
    global _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = _build.MODEL_LIB_PATH
        if not os.path.exists(path):
            raise NativeLibraryMissing(
                "%s not found. Build it with `python -m returnn_amd.build` (needs hipcc; cross-compiles for gfx950 without a GPU)." % path
            )
        lib = ctypes.CDLL(path)
        abi = int(lib.rtn_model_ops_abi_version())
        if abi != EXPECTED_ABI:
            raise NativeLibraryMismatch(
                "%s reports ABI version %i, this binding is written for %i: rebuild it with `python -m returnn_amd.build`" % (path, abi, EXPECTED_ABI)
            )
        vp, i32, i64, f32, sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
        lib.rtn_model_ops_last_error.restype = ctypes.c_char_p
        lib.rtn_model_ops_last_error.argtypes = []
        sizes = [i64, i32, i32, i32, i32, i32, i32]
        lib.rtn_delta_rule_fwd_workspace_bytes.restype, lib.rtn_delta_rule_fwd_workspace_bytes.argtypes = sz, sizes + [i32]
        lib.rtn_delta_rule_saved_bytes.restype, lib.rtn_delta_rule_saved_bytes.argtypes = sz, sizes
        lib.rtn_delta_rule_fwd.argtypes = [vp, i64, vp, i64, vp, i64, vp, vp, vp, vp, vp, vp, vp] + sizes + [f32, i32, vp, sz, vp]
        lib.rtn_delta_rule_bwd_workspace_bytes.restype, lib.rtn_delta_rule_bwd_workspace_bytes.argtypes = sz, sizes
        lib.rtn_delta_rule_bwd.argtypes = [vp, i64, vp, i64, vp, i64, vp, vp, vp, vp, vp, i64, vp, vp, vp, vp, vp, vp, vp] + sizes + [f32, i32, vp, sz, vp]
        lib.rtn_embedding_fwd.argtypes = [vp, vp, i64, vp, i64, i64, i64, i32, f32, vp]
        lib.rtn_embedding_bwd_workspace_bytes.restype, lib.rtn_embedding_bwd_workspace_bytes.argtypes = sz, [i64, i64, i64, i32]
        lib.rtn_embedding_bwd.argtypes = [vp, vp, i64, vp, i64, i64, i64, i32, f32, vp, sz, vp]
        lib.rtn_beam_select_workspace_bytes.restype, lib.rtn_beam_select_workspace_bytes.argtypes = sz, [i32, i32, i64, i32, i32]
        lib.rtn_beam_select.argtypes = [vp, i64, vp, vp, i64, vp, vp, vp, i32, i32, i64, i32, i32, vp, sz, vp]
        lib.rtn_reorder_rows.argtypes = [i32, vp, vp, vp, vp, i32, i32, i32, vp]
        _lib = lib
        return lib


def last_error() -> str:
    return load().rtn_model_ops_last_error().decode("utf8", "replace")


def native():
    """The torch side of the calls, given the library's entry points: loaded once, never built here, no fallback."""
    global _native_module
    if _native_module is not None:
        return _native_module
    with _lock:
        if _native_module is None:
            import torch  # noqa: F401 (whose libraries the binding is linked against)

            lib = load()
            try:
                from . import _rtn_model
            except ImportError as exc:
                raise NativeLibraryMissing("the torch binding could not be loaded (%s).  Build it with `python -m returnn_amd.build`." % exc) from exc
            _rtn_model.init({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in SYMBOLS})
            _native_module = _rtn_model
    return _native_module
