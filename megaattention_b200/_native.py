"""The operators' native calls (``csrc/calls.cpp``), built for the torch that is installed and bound to the
library's entry points: ``calls``, loaded when it is first used, so that what does without it (the fused path)
can be imported where it cannot be built.  There is no fallback: without the module its use raises ImportError.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import os

import torch

from . import _cabi, build as _build


def _load():
    if _build._stale(_build.LIB_CALLS):
        try:
            _build.build_calls()
        except Exception as exc:  # no compiler on this machine: use what is there, if anything
            if not os.path.exists(_build.LIB_CALLS):
                raise ImportError(f"{os.path.basename(_build.LIB_CALLS)} is missing and cannot be built: {exc}")
    spec = importlib.util.spec_from_file_location(f"{__package__}._calls", _build.LIB_CALLS)
    _calls = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(_calls)
    if _calls.torch_version != torch.__version__:
        raise ImportError(f"{os.path.basename(_build.LIB_CALLS)} was built for torch {_calls.torch_version}, this is "
                          f"{torch.__version__}: delete it")
    _calls.bind(*(C.cast(getattr(_cabi.lib, name), C.c_void_p).value for name in (
        "ma_rmsnorm_quant", "ma_linear_quant", "ma_dequant", "ma_rope_append", "ma_strerror")))
    return _calls


def __getattr__(name):
    if name != "calls":
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    module = globals()["calls"] = _load()
    globals().pop("__getattr__", None)         # (a look-up in a module that has one takes four times as long)
    return module
