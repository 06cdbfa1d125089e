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

from .. import _cabi
from ._call import BF16, F32, I8, on_device, packer, pitch_of, queue

_OUT = {BF16: 0, F32: 1}
_pack = packer(_cabi.LinearQuantArgs)
_fn = _cabi.lib.ma_linear_quant
_pack_dequant = packer(_cabi.DequantArgs)


def _output(out, rows, n, dtype, dev):
    """The output, its row pitch and whether it is fp32."""
    if out is None:
        assert dtype in _OUT, "bf16 or fp32"
        return torch.empty(rows, n, dtype=dtype, device=dev), n, _OUT[dtype]
    assert out.shape == (rows, n) and out.dtype in _OUT and out.device == dev, "out: [rows, columns] bf16 or fp32"
    pitch, one = out.stride()
    assert (one == 1 or n <= 1) and (pitch >= n or rows <= 1), "out: columns next to each other, no rows that overlap"
    return out, pitch if rows > 1 else n, _OUT[out.dtype]


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
    ``[tokens, out]`` in ``out_dtype`` (bf16 or fp32), or fills ``out`` (any row pitch).  Queued on the
    current stream of that device."""
    shape, strides, at = x.shape, x.stride(), x.data_ptr()
    w_shape, w_strides, w_at = weight.shape, weight.stride(), weight.data_ptr()
    dev = x.device
    index = dev.index
    assert len(shape) == 2 == len(w_shape) and shape[1] == w_shape[1] > 0, "x [tokens, in] and weight [out, in]"
    assert x.dtype is I8 is weight.dtype and x.is_cuda and weight.get_device() == index, "int8 on one CUDA device"
    pitch, w_pitch = pitch_of(strides, shape), pitch_of(w_strides, w_shape)
    assert not (at | pitch | w_at | w_pitch) & 15 and (strides[1] == 1 == w_strides[1] or shape[1] == 1), \
        "rows must start at multiples of 16 bytes, columns next to each other"
    tokens, inner = shape
    width = w_shape[0]
    assert x_scale.shape == (tokens,) and x_scale.dtype is F32 and x_scale.get_device() == index and \
        x_scale.is_contiguous(), "x_scale: [tokens] fp32"
    assert weight_scale.shape == (width,) and weight_scale.dtype is F32 and weight_scale.get_device() == index and \
        weight_scale.is_contiguous(), "weight_scale: [out] fp32"
    b_at = 0
    if bias is not None:
        assert bias.shape == (width,) and bias.dtype is BF16 and bias.get_device() == index and bias.is_contiguous(), \
            "bias: [out] bf16"
        b_at = bias.data_ptr()
    out, out_pitch, f32 = _output(out, tokens, width, out_dtype, dev)
    if tokens and width:
        queue(_fn, _pack(at, w_at, x_scale.data_ptr(), weight_scale.data_ptr(), b_at, out.data_ptr(), pitch, w_pitch,
                         out_pitch, tokens, inner, width, f32), index, "ma_linear_quant")
    return out


def dequantize_int8(q, scale, *, out=None, out_dtype=torch.bfloat16):
    """``q [rows, n]`` int8 with rows at multiples of 16 bytes as the values it stands for, ``q * scale[:,
    None]``, rounded once to ``out_dtype`` (bf16 or fp32): an 8-bit weight for what reads 16 bits, as
    ``FusedPrefillLayer(ws, dequantize_int8(W_o, W_o_scale).T)``, or an 8-bit activation beside it.  Queued on
    the current stream of the device."""
    shape, strides, at = q.shape, q.stride(), q.data_ptr()
    dev = q.device
    assert len(shape) == 2 and q.dtype is I8 and q.is_cuda, "q: [rows, n] int8 on a CUDA device"
    pitch = pitch_of(strides, shape)
    rows, n = shape
    assert not (at | pitch) & 15 and (strides[1] == 1 or n <= 1), \
        "q: rows must start at multiples of 16 bytes, columns next to each other"
    assert scale.shape == (rows,) and scale.dtype is F32 and scale.device == dev and scale.is_contiguous()
    out, out_pitch, f32 = _output(out, rows, n, out_dtype, dev)
    if rows and n:
        queue(_cabi.lib.ma_dequant, _pack_dequant(at, scale.data_ptr(), out.data_ptr(), pitch, out_pitch, rows, n, f32,
                                                  0), dev.index, "ma_dequant")
    return out


def check_linear_status(device=None):
    """Synchronise the device's current stream and raise if a device-side wait of ``linear_int8`` gave
    up since the last check (the output of such a call is undefined)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    st = _cabi.Status()
    with on_device(dev):
        rc = _cabi.lib.ma_linear_status(torch.cuda.current_stream(dev).cuda_stream, C.byref(st))
    if rc != _cabi.MA_OK:
        raise RuntimeError(f"linear_int8: {_cabi.strerror(rc)} (code={st.code} site=0x{st.site:x} "
                           f"cta={st.cta} aux={st.aux})")
