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
from ._call import queue
from .rope import default_inv_freq


def _heads(t, dev, what):
    assert t.dim() == 3 and t.shape[2] == 128 and t.dtype == torch.bfloat16 and t.device == dev, \
        f"{what}: [tokens, heads, 128] bf16 on {dev}"
    tok, head, one = t.stride()
    assert one == 1 and t.data_ptr() % 16 == 0 and tok % 8 == 0 and head % 8 == 0 and tok >= 0 and head >= 0, \
        f"{what}: heads must start at multiples of 16 bytes"
    return tok, head


def _words(t, dim, dev, what):
    assert torch.is_tensor(t) and t.dtype == torch.int32 and t.dim() == dim and t.device == dev, \
        f"{what}: int32 on {dev}"
    assert t.stride(-1) == 1 or t.shape[-1] <= 1, f"{what}: columns must be next to each other"
    return t


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
    assert q.is_cuda
    sq, sk, sv = _heads(q, dev, "q"), _heads(k, dev, "k"), _heads(v, dev, "v")
    tokens, H = q.shape[:2]
    Hkv = k.shape[1]
    assert H and Hkv and k.shape == v.shape and k.shape[0] == tokens, "q [tokens, H, 128]; k, v [tokens, H_kv, 128]"
    for c in (k_cache, v_cache):
        assert c.dtype == torch.bfloat16 and c.device == dev and c.is_contiguous() and c.data_ptr() % 16 == 0
        assert c.shape[-2:] == (Hkv, 128) and (c.dim() == 3 and c.shape[0] % 128 == 0 or
                                               c.dim() == 4 and c.shape[1] == 128), \
            "caches: [num_pages, 128, H_kv, 128] or [num_pages * 128, H_kv, 128]"
    pages = k_cache.shape[0] if k_cache.dim() == 4 else k_cache.shape[0] // 128
    assert pages and k_cache.shape == v_cache.shape
    _words(page_table, 2, dev, "page_table")
    _words(cache_seqlens, 1, dev, "cache_seqlens")
    _words(cu_seqlens_q, 1, dev, "cu_seqlens_q")
    batch, width = page_table.shape
    assert batch and width and cache_seqlens.shape[0] == batch and cu_seqlens_q.shape[0] == batch + 1
    w = default_inv_freq(theta, dev) if inv_freq is None else inv_freq
    assert w.shape == (64,) and w.dtype == torch.float32 and w.device == dev and w.is_contiguous()
    if out is None:
        out = torch.empty(tokens, H, 128, dtype=torch.bfloat16, device=dev)
        so = (H * 128, 128)
    else:
        so = _heads(out, dev, "out")
        assert out.shape == q.shape
    if dropped is not None:
        assert dropped.shape == (1,) and dropped.dtype == torch.int32 and dropped.device == dev
    if tokens:
        a = _cabi.RopeAppendArgs(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            cu_seqlens_q.data_ptr(), cache_seqlens.data_ptr(), page_table.data_ptr(), w.data_ptr(),
            0 if dropped is None else dropped.data_ptr(), *sq, *sk, *sv, *so,
            page_table.stride(0) if batch > 1 else width, tokens, batch, H, Hkv, pages, width)
        queue(_cabi.lib.ma_rope_append, a, dev, "ma_rope_append")
    return out          # (a w made here was allocated on this stream: reuse after free is stream-ordered)
