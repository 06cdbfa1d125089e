"""Residual add + RMSNorm with an 8-bit result: integers and one scale per token, as
``linear_int8`` reads them.

The 8-bit form of ``residual_rmsnorm``, for layers whose next projection runs in 8-bit integers (the
reference lists a "residual / RMSNorm consumer" as its next step, README.md:41-44 of the reference, and has
no code for it).  One HBM-bound CUDA kernel behind the C ABI (``ma_rmsnorm_quant``), from packed rows or
straight from the fused launch's tile-padded output::

    q, scale, residual = residual_rmsnorm_int8(ws, residual, weight, eps=1e-6, inplace=True)
    qkv = linear_int8(q, scale, W_qkv, W_scale)

    q, scale = rmsnorm_int8(x, weight)                              # a model's first norm
    q, scale, residual = rmsnorm_int8(y, weight, residual=residual) # behind another projection

``h = bf16(x + residual)``, ``y = h * rsqrt(mean(h^2) + eps) * weight``, ``scale = max|y| / 127`` per
token and ``q = round(y / scale)`` with the statistics in fp32.  A row of zeros gets scale 0 and zeros, a
row that is not finite scale NaN and zeros.  ``q``'s rows start at multiples of 16 bytes (what the matrix
product loads them by): of a ``hidden`` that is not a multiple of 16 it is a view with a longer row pitch.
"""
from __future__ import annotations

import torch

from .. import _cabi
from ._call import BF16, F32, I8, packer, pitch_of, queue

_pack = packer(_cabi.RmsNormQuantArgs)
_fn = _cabi.lib.ma_rmsnorm_quant


def _queue(x, x_pitch, tokens, rows, hidden, weight, eps, residual, inplace, out, scale, dev, tiles, stream):
    at = dev.index
    w = weight.data_ptr()
    assert weight.shape == (hidden,) and weight.dtype is BF16 and weight.get_device() == at and \
        weight.is_contiguous() and not w & 15, "weight: [hidden] bf16, 16-byte aligned"
    assert not hidden & 7 and 0 < hidden <= 16384, "hidden: a multiple of 8, up to 16384"
    if out is None:
        q_pitch = (hidden + 15) & ~15
        q = torch.empty(tokens, q_pitch, dtype=I8, device=dev)
        q_at = q.data_ptr()
        if q_pitch != hidden:
            q = q[:, :hidden]
    else:
        q, q_at, strides = out, out.data_ptr(), out.stride()
        assert q.shape == (tokens, hidden) and q.dtype is I8 and q.get_device() == at and strides[1] == 1
        q_pitch = pitch_of(strides, q.shape)
        assert not (q_at | q_pitch) & 15, "out: rows must start at multiples of 16 bytes"
    if scale is None:
        scale = torch.empty(tokens, dtype=F32, device=dev)
    else:
        assert scale.shape == (tokens,) and scale.dtype is F32 and scale.get_device() == at and scale.is_contiguous()
    new_res, r_in, r_out, r_pitch, n_pitch = None, 0, 0, 0, 0
    if residual is not None:
        r_in, strides = residual.data_ptr(), residual.stride()
        assert residual.shape == (tokens, hidden) and residual.dtype is BF16 and residual.get_device() == at, \
            "residual: [tokens, hidden] bf16 on the device of x"
        r_pitch = pitch_of(strides, residual.shape)
        assert strides[1] == 1 and not r_in & 15 and not r_pitch & 7, \
            "residual: rows must start at multiples of 16 bytes, columns next to each other"
        if inplace:
            new_res, n_pitch = residual, r_pitch
        else:
            new_res, n_pitch = torch.empty_like(residual, memory_format=torch.contiguous_format), hidden
        r_out = new_res.data_ptr()
    if tokens:
        queue(_fn, _pack(x, r_in, w, r_out, q_at, scale.data_ptr(), *tiles, x_pitch, r_pitch, n_pitch, q_pitch, rows,
                         hidden, eps, 0), at, "ma_rmsnorm_quant", stream)
    return (q, scale) if residual is None else (q, scale, new_res)


def rmsnorm_int8(x, weight, eps: float = 1e-6, *, residual=None, inplace: bool = False, out=None, scale=None):
    """``x [tokens, hidden]``, ``weight [hidden]`` and, if given, ``residual [tokens, hidden]`` bf16 on
    one CUDA device; rows at multiples of 16 bytes, ``hidden`` a multiple of 8 up to 16384.  Returns
    ``(q [tokens, hidden] int8, scale [tokens] fp32)``, and the new residual stream as a third where there is a
    residual (with ``inplace`` it is updated where it is).  ``out`` and ``scale`` take the results.
    Queued on the current stream of that device."""
    shape, strides, at = x.shape, x.stride(), x.data_ptr()
    assert len(shape) == 2 and x.dtype is BF16 and x.is_cuda, "x: [tokens, hidden] bf16 on a CUDA device"
    pitch = pitch_of(strides, shape)
    assert strides[1] == 1 and not at & 15 and not pitch & 7, \
        "x: rows must start at multiples of 16 bytes, columns next to each other"
    assert residual is not None or not inplace, "inplace needs a residual"
    return _queue(at, pitch, shape[0], shape[0], shape[1], weight, eps, residual, inplace, out, scale, x.device,
                  (0, 0, 0), None)


def residual_rmsnorm_int8(ws, residual, weight, eps: float = 1e-6, *, inplace: bool = False, out=None, scale=None,
                          meta=None):
    """The same on the fused launch's output, read in place from ``ws.csym``: returns ``(q, scale,
    new_residual)``.  Queued on the workspace's stream behind the launch, as ``residual_rmsnorm`` is."""
    meta = meta if meta is not None else ws._meta
    assert meta is not None, "no layer has been set on this workspace"
    tokens = int(meta.cu_seqlens_q[-1])
    tiles = (ws.cu_q.data_ptr(), ws.fa_b.data_ptr(), ws.fa_mb.data_ptr())
    assert residual is not None
    with ws._on_stream():                  # (the results' memory is the workspace's stream's too)
        return _queue(ws.csym.data_ptr(), ws.num_out * 128, tokens, int(meta.num_row_tiles), ws.hidden, weight, eps,
                      residual, inplace, out, scale, ws.dev, tiles, ws._stream().cuda_stream)
