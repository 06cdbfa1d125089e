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

from .. import _native
from .rope import default_inv_freq


def rope_append(q, k, v, k_cache, v_cache, page_table, cache_seqlens, cu_seqlens_q, *, theta: float = 10000.0,
                inv_freq=None, out=None, dropped=None):
    """``q [tokens, H, 128]``, ``k, v [tokens, H_kv, 128]`` bf16 (any strides that keep heads at multiples
    of 16 bytes); ``k_cache, v_cache`` bf16, contiguous, ``[num_pages, 128, H_kv, 128]`` or token pools
    ``[num_pages * 128, H_kv, 128]``; ``page_table [batch, pages]``, ``cache_seqlens [batch]`` and
    ``cu_seqlens_q [batch + 1]`` (ascending from 0; sequences may be empty) int32; all on one CUDA device.  Returns
    the rotated q, contiguous, or in ``out``: ``q`` itself, or memory that is no part of q, k and v (where it lies
    between their tokens, its own are as far apart as theirs).

    Rows from ``cu_seqlens_q[-1]`` on are left as they are (in a new output: undefined).  A row whose
    page is not in the table or not in the cache is not appended; one that would lie before its
    sequence's first key is passed over; ``dropped`` (int32 ``[1]``, on the device) is added the number of
    both.  Two rows must not have the same place in the cache, nor a row's place be where another's k or v lies.
    ``inv_freq [64]`` fp32 takes the place of ``theta``.  Queued on the current stream of the device."""
    if inv_freq is None:      # (allocated on this stream: reuse after free is stream-ordered)
        inv_freq = default_inv_freq(theta, q.device)
    return _native.calls.rope_append(q, k, v, k_cache, v_cache, page_table, cache_seqlens, cu_seqlens_q, inv_freq, out, dropped)
