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
row that is not finite (or its sum of squares) scale NaN and zeros.  With an ``eps`` of 0, or close to it, so does a
row whose ``mean(h^2) + eps`` is below 2^-126, where fp32 squares lose their bits; ``h * weight`` below 1.6e-36
throughout counts as zeros.  ``q``'s rows start at multiples of 16 bytes (what the matrix
product loads them by): of a ``hidden`` that is not a multiple of 16 it is a view with a longer row pitch.
"""
from __future__ import annotations

from .. import _native


def rmsnorm_int8(x, weight, eps: float = 1e-6, *, residual=None, inplace: bool = False, out=None, scale=None):
    """``x [tokens, hidden]``, ``weight [hidden]`` and, if given, ``residual [tokens, hidden]`` bf16 on
    one CUDA device; rows at multiples of 16 bytes, ``hidden`` a multiple of 8 up to 16384.  Returns
    ``(q [tokens, hidden] int8, scale [tokens] fp32)``, and the new residual stream as a third where there is a
    residual (with ``inplace`` it is updated where it is).  ``out`` and ``scale`` take the results; they and an
    updated residual share no memory with each other or an input, except that ``out``'s rows may lie in ``x``'s (row
    for row) and that the residual may be ``x``.
    Queued on the current stream of that device."""
    return _native.calls.rmsnorm_int8(x, weight, eps, residual, inplace, out, scale, None)


def residual_rmsnorm_int8(ws, residual, weight, eps: float = 1e-6, *, inplace: bool = False, out=None, scale=None,
                          meta=None):
    """The same on the fused launch's output, read in place from ``ws.csym``: returns ``(q, scale,
    new_residual)``.  Queued on the workspace's stream behind the launch, as ``residual_rmsnorm`` is."""
    meta = meta if meta is not None else ws._meta
    assert meta is not None, "no layer has been set on this workspace"
    assert residual is not None
    tiles = (ws.cu_q.data_ptr(), ws.fa_b.data_ptr(), ws.fa_mb.data_ptr(), int(meta.num_row_tiles),
             int(meta.cu_seqlens_q[-1]), ws.hidden, ws.num_out * 128, ws._stream().cuda_stream)
    with ws._on_stream():                  # (the results' memory is the workspace's stream's too)
        return _native.calls.rmsnorm_int8(ws.csym, weight, eps, residual, inplace, out, scale, tiles)
