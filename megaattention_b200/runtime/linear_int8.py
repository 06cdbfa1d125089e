"""Matrix product of 8-bit integers with a scale for each token and each output channel.

The projections either side of the attention path in their 8-bit form: the reference names a "QKV-proj"
producer as a step it has not built (README.md:41-44 of the reference).  One CUDA kernel behind the C ABI
(``ma_linear_quant``) on the integer tensor path::

    W, W_scale = quantize_weight_int8(linear.weight)       # once: [out_features, in_features]
    q, scale = rmsnorm_int8(x, norm_weight)
    y = linear_int8(q, scale, W, W_scale, bias=linear.bias)

``y[m, n] = (sum_k x[m, k] * weight[n, k]) * x_scale[m] * weight_scale[n] + bias[n]``: the sum exact in
32-bit integers, the rest in fp32, rounded once.
"""
from __future__ import annotations

import ctypes as C

import torch

from .. import _cabi, _native


def quantize_weight_int8(weight):
    """``weight [out_features, in_features]`` (floating point) as ``(int8, scale [out_features] fp32)``, a
    scale per row; rows at multiples of 16 bytes, as ``linear_int8`` wants them.  Done once, when a model is
    loaded, in plain torch operations."""
    assert weight.dim() == 2 and weight.is_floating_point()
    n, k = weight.shape
    w = weight.float()
    top = w.abs().amax(dim=1, keepdim=True)
    q = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=weight.device)
    q[:, :k] = torch.where(top > 0, torch.round(w / top * 127.0), w)
    return q[:, :k], (top / 127.0).reshape(n)


def linear_int8(x, x_scale, weight, weight_scale, *, bias=None, out=None, out_dtype=torch.bfloat16):
    """``x [tokens, in]`` and ``weight [out, in]`` int8 with rows at multiples of 16 bytes (as
    ``rmsnorm_int8`` and ``quantize_weight_int8`` make them), ``x_scale [tokens]`` and ``weight_scale
    [out]`` fp32, ``bias [out]`` bf16 or none, all on one CUDA device; ``in`` up to 131071.  Returns
    ``[tokens, out]`` in ``out_dtype`` (bf16 or fp32), or fills ``out`` (any row pitch; no memory of the inputs).
    Queued on the current stream of that device."""
    return _native.calls.linear_int8(x, x_scale, weight, weight_scale, bias, out, out_dtype)


def dequantize_int8(q, scale, *, out=None, out_dtype=torch.bfloat16):
    """``q [rows, n]`` int8 with rows at multiples of 16 bytes as the values it stands for, ``q * scale[:,
    None]``, rounded once to ``out_dtype`` (bf16 or fp32): an 8-bit weight for what reads 16 bits, as
    ``FusedPrefillLayer(ws, dequantize_int8(W_o, W_o_scale).T)``, or an 8-bit activation beside it.  Queued on
    the current stream of the device."""
    return _native.calls.dequantize_int8(q, scale, out, out_dtype)


def check_linear_status(device=None):
    """Synchronise the device's current stream and raise if a device-side wait of ``linear_int8`` on that device
    gave up since the last check, on whichever stream: one check raises, the first (what such a call did not
    compute is NaN)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    st = _cabi.Status()
    with torch.cuda.device(dev):
        rc = _cabi.lib.ma_linear_status(torch.cuda.current_stream(dev).cuda_stream, C.byref(st))
    if rc != _cabi.MA_OK:
        raise RuntimeError(f"linear_int8: {_cabi.strerror(rc)} (code={st.code} site=0x{st.site:x} "
                           f"cta={st.cta} aux={st.aux})")
