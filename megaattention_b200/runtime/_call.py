"""What the operators' calls share.  Small calls take as long as their host side does, so it is short: an
attribute of a tensor is read once, dtypes are compared by identity, arguments are packed in one go."""
from __future__ import annotations

import contextlib
import ctypes
import struct

import torch

from .. import _cabi

BF16, F32, I32, I8 = torch.bfloat16, torch.float32, torch.int32, torch.int8
_get_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_CODES = {"c_ulong": "Q", "c_long": "q", "c_int": "i", "c_float": "f", "c_uint": "I"}


def packer(structure):
    """The bytes of a C-ABI structure from its fields in order."""
    code = struct.Struct("=" + "".join(_CODES[t.__name__] for _, t in structure._fields_))
    assert code.size == ctypes.sizeof(structure), "no padding between the fields"
    return code.pack


def on_device(dev):
    """``torch.cuda.device(dev)``, or nothing to do if that is current."""
    if _get_device() == dev.index:
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def queue(fn, args, device, what, stream=None):
    """One C call with packed ``args`` on ``stream`` (default: the current one of device number
    ``device``), with that device current."""
    if stream is None:
        stream = _raw_stream(device)
    if _get_device() == device:
        rc = fn(args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(args, stream)
    if rc:
        _cabi.check(rc, what)


def pitch_of(strides, shape):
    """Elements from one row to the next (of a single row: its length, up to a multiple of 16)."""
    return strides[0] if shape[0] > 1 else (shape[1] + 15) // 16 * 16
