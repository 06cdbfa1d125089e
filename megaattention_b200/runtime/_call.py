"""What the operators' calls share: the stream and the device that a call is queued on."""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from .. import _cabi


def on_device(dev):
    """``torch.cuda.device(dev)``, or nothing to do if that is current."""
    if torch._C._cuda_getDevice() == dev.index:
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def queue(fn, args, dev, what, stream=None):
    """One C call on ``stream`` (default: the current one of ``dev``), with ``dev`` current."""
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(dev.index)
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(C.addressof(args), stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(C.addressof(args), stream)
    if rc != _cabi.MA_OK:
        _cabi.check(rc, what)


def rows_of(t, dtype, dev, align, what):
    """``t`` is ``[rows, n]`` of ``dtype`` on ``dev`` with columns next to each other and rows that start
    ``align`` bytes apart or a multiple of it."""
    assert t.dim() == 2 and t.dtype == dtype and t.device == dev, f"{what}: [rows, columns] {dtype} on {dev}"
    assert t.stride(1) == 1 or t.shape[1] <= 1, f"{what}: columns must be next to each other"
    assert t.data_ptr() % align == 0 and pitch_of(t) * t.element_size() % align == 0, \
        f"{what}: rows must start at multiples of {align} bytes"
    return t


def pitch_of(t):
    """Elements from one row to the next (of a single row: its length, up to a multiple of 16)."""
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 16) * 16
