"""Rotary position embedding of a step's queries and new keys, with keys and values appended to
the paged KV cache on the way: the producer of a paged ``FusedPrefillLayer``.

``rope_qk_`` rotates keys that lie packed; a paged layer reads its keys from pages.  One HBM-bound CUDA
kernel behind the C ABI (``ma_rope_append``) takes the projection's output as it is - q, k and v may be
strided views of one tensor - and leaves what the layer reads (the reference lists the producer as a
step it has not built, README.md:41-44 of the reference)::

    qkv = linear_int8(x, x_scale, W_qkv, W_scale)                       # [tokens, (H + 2 H_kv) * 128]
    q, k, v = (t.unflatten(1, (-1, 128)) for t in qkv.split([H * 128, H_kv * 128, H_kv * 128], dim=1))
    q = rope_append(q, k, v, k_cache, v_cache, page_table, cache_seqlens, cu_seqlens_q_device, inv_freq=inv_freq)
    layer(q, k_cache, v_cache, cu_seqlens_q, page_table=page_table, cache_seqlens=cache_seqlens)

Row ``t`` of sequence ``b`` has position ``cache_seqlens[b] - (cu_seqlens_q[b + 1] - t)`` (the lengths
count the new keys, as the layer's do).  Everything is read on the device and nothing waits for the
host, so a captured call follows the arrays' contents.
"""
from __future__ import annotations

import torch

from .. import _cabi
from ._call import BF16, F32, I32, packer, queue
from .rope import default_inv_freq

_pack = packer(_cabi.RopeAppendArgs)
_fn = _cabi.lib.ma_rope_append


def rope_append(q, k, v, k_cache, v_cache, page_table, cache_seqlens, cu_seqlens_q, *, theta: float = 10000.0,
                inv_freq=None, out=None, dropped=None):
    """``q [tokens, H, 128]``, ``k, v [tokens, H_kv, 128]`` bf16 (any strides that keep heads at multiples
    of 16 bytes); ``k_cache, v_cache`` bf16, contiguous, ``[num_pages, 128, H_kv, 128]`` or token pools
    ``[num_pages * 128, H_kv, 128]``; ``page_table [batch, pages]``, ``cache_seqlens [batch]`` and
    ``cu_seqlens_q [batch + 1]`` (ascending from 0; sequences may be empty) int32; all on one CUDA device.  Returns
    the rotated q, contiguous, or in ``out`` (which may be ``q`` itself).

    Rows from ``cu_seqlens_q[-1]`` on are left as they are (in a new output: undefined).  A row whose
    page is not in the table or not in the cache is not appended; one that would lie before its
    sequence's first key is passed over; ``dropped`` (int32 ``[1]``, on the device) is added the number of
    both.  Two rows must not have the same place in the cache.  ``inv_freq [64]`` fp32 takes the place of
    ``theta``.  Queued on the current stream of the device."""
    dev = q.device
    at = dev.index
    shape, kv, cache = q.shape, k.shape, k_cache.shape
    tokens, H, d = shape
    Hkv = kv[1]
    assert d == 128 == kv[2] and kv == v.shape and kv[0] == tokens and H and Hkv, \
        "q [tokens, H, 128]; k, v [tokens, H_kv, 128]"
    assert q.dtype is BF16 is k.dtype and BF16 is v.dtype is k_cache.dtype and v_cache.dtype is BF16, "bf16"
    assert q.is_cuda and k.get_device() == at == v.get_device() and k_cache.get_device() == at == v_cache.get_device(), \
        "one CUDA device"
    assert cache == v_cache.shape and cache[-1] == 128 and cache[-2] == Hkv and (
        len(cache) == 4 and cache[1] == 128 or len(cache) == 3 and not cache[0] & 127) and cache[0] and \
        k_cache.is_contiguous() and v_cache.is_contiguous(), \
        "caches: contiguous, [num_pages, 128, H_kv, 128] or [num_pages * 128, H_kv, 128]"
    pages = cache[0] if len(cache) == 4 else cache[0] >> 7
    q_tok, q_head, q_one = q.stride()
    k_tok, k_head, k_one = k.stride()
    v_tok, v_head, v_one = v.stride()
    q_at, k_at, v_at = q.data_ptr(), k.data_ptr(), v.data_ptr()
    kc_at, vc_at = k_cache.data_ptr(), v_cache.data_ptr()
    assert q_one == 1 == k_one == v_one and not (q_at | k_at | v_at | kc_at | vc_at) & 15 and \
        not (q_tok | q_head | k_tok | k_head | v_tok | v_head) & 7, "heads must start at multiples of 16 bytes"
    batch, width = page_table.shape
    assert batch and width and cache_seqlens.shape == (batch,) and cu_seqlens_q.shape == (batch + 1,), \
        "page_table [batch, pages], cache_seqlens [batch], cu_seqlens_q [batch + 1]"
    assert page_table.dtype is I32 is cache_seqlens.dtype and cu_seqlens_q.dtype is I32, "page_table and lengths: int32"
    assert page_table.get_device() == at == cache_seqlens.get_device() and cu_seqlens_q.get_device() == at, \
        "page_table and lengths: on the device of q"
    t_pitch, t_one = page_table.stride()
    assert (t_one == 1 or width == 1) and cache_seqlens.is_contiguous() and cu_seqlens_q.is_contiguous(), \
        "page_table and lengths: columns next to each other"
    w = default_inv_freq(theta, dev) if inv_freq is None else inv_freq
    assert w.shape == (64,) and w.dtype is F32 and w.get_device() == at and w.is_contiguous(), "inv_freq: [64] fp32"
    if out is None:
        out = torch.empty(tokens, H, 128, dtype=BF16, device=dev)
        o_at, o_tok, o_head = out.data_ptr(), H * 128, 128
    else:
        o_at = out.data_ptr()
        o_tok, o_head, o_one = out.stride()
        assert out.shape == shape and out.dtype is BF16 and out.get_device() == at and o_one == 1 and \
            not o_at & 15 and not (o_tok | o_head) & 7, "out: as q"
        assert (o_tok >= 128 or tokens == 1) and (o_head >= 128 or H == 1), "heads of out overlap"
    d_at = 0
    if dropped is not None:
        assert dropped.shape == (1,) and dropped.dtype is I32 and dropped.get_device() == at, "dropped: [1] int32"
        d_at = dropped.data_ptr()
    if tokens:
        queue(_fn, _pack(q_at, k_at, v_at, o_at, kc_at, vc_at, cu_seqlens_q.data_ptr(), cache_seqlens.data_ptr(),
                         page_table.data_ptr(), w.data_ptr(), d_at, q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok,
                         o_head, t_pitch if batch > 1 else width, tokens, batch, H, Hkv, pages, width), at,
              "ma_rope_append")
    return out          # (a w made here was allocated on this stream: reuse after free is stream-ordered)
