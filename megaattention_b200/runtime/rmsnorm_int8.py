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
from ._call import pitch_of, queue, rows_of


def _eight_bit_rows(rows, hidden, dev, out):
    if out is None:
        pitch = (hidden + 15) // 16 * 16
        out = torch.empty(rows, pitch, dtype=torch.int8, device=dev)
        return out if pitch == hidden else out[:, :hidden]
    rows_of(out, torch.int8, dev, 16, "out")
    assert out.shape == (rows, hidden)
    return out


def _queue(x, x_pitch, tokens, rows, hidden, weight, eps, residual, inplace, out, scale, dev, tiles, stream):
    assert weight.shape == (hidden,) and weight.dtype == torch.bfloat16 and weight.device == dev
    assert weight.is_contiguous() and weight.data_ptr() % 16 == 0
    assert hidden % 8 == 0 and 0 < hidden <= 16384, "hidden: a multiple of 8, up to 16384"
    q = _eight_bit_rows(tokens, hidden, dev, out)
    if scale is None:
        scale = torch.empty(tokens, dtype=torch.float32, device=dev)
    assert scale.shape == (tokens,) and scale.dtype == torch.float32 and scale.device == dev
    assert scale.is_contiguous()
    new_res, res = None, (0, 0, 0, 0)
    if residual is not None:
        rows_of(residual, torch.bfloat16, dev, 16, "residual")
        assert residual.shape == (tokens, hidden)
        new_res = residual if inplace else torch.empty(tokens, hidden, dtype=torch.bfloat16, device=dev)
        res = (residual.data_ptr(), new_res.data_ptr(), pitch_of(residual), pitch_of(new_res))
    if tokens:
        a = _cabi.RmsNormQuantArgs(x, res[0], weight.data_ptr(), res[1], q.data_ptr(), scale.data_ptr(), *tiles,
                                   x_pitch, res[2], res[3], pitch_of(q), rows, hidden, eps, 0)
        queue(_cabi.lib.ma_rmsnorm_quant, a, dev, "ma_rmsnorm_quant", stream)
    return (q, scale) if residual is None else (q, scale, new_res)


def rmsnorm_int8(x, weight, eps: float = 1e-6, *, residual=None, inplace: bool = False, out=None, scale=None):
    """``x [tokens, hidden]``, ``weight [hidden]`` and, if given, ``residual [tokens, hidden]`` bf16 on
    one CUDA device; rows at multiples of 16 bytes, ``hidden`` a multiple of 8 up to 16384.  Returns
    ``(q [tokens, hidden] int8, scale [tokens] fp32)``, and the new residual stream as a third where there is a
    residual (with ``inplace`` it is updated where it is).  ``out`` and ``scale`` take the results.
    Queued on the current stream of that device."""
    dev = x.device
    assert x.is_cuda
    rows_of(x, torch.bfloat16, dev, 16, "x")
    assert residual is not None or not inplace, "inplace needs a residual"
    tokens, hidden = x.shape
    return _queue(x.data_ptr(), pitch_of(x), tokens, tokens, hidden, weight, eps, residual, inplace, out, scale, dev,
                  (0, 0, 0), None)


def residual_rmsnorm_int8(ws, residual, weight, eps: float = 1e-6, *, inplace: bool = False, out=None, scale=None,
                          meta=None):
    """The same on the fused launch's output, read in place from ``ws.csym``: returns ``(q, scale,
    new_residual)``.  Queued on the workspace's stream behind the launch, as ``residual_rmsnorm`` is."""
    meta = meta if meta is not None else ws._meta
    assert meta is not None, "no layer has been set on this workspace"
    tokens = int(meta.cu_seqlens_q[-1])
    tiles = (ws.cu_q.data_ptr(), ws.fa_b.data_ptr(), ws.fa_mb.data_ptr())
    return _queue(ws.csym.data_ptr(), ws.num_out * 128, tokens, int(meta.num_row_tiles), ws.hidden, weight, eps,
                  residual, inplace, out, scale, ws.dev, tiles, ws._stream().cuda_stream)
