"""Statements in float64 of the operators between two layers (TEST INFRASTRUCTURE: imported by tests
only, never by the product path): the norm with an 8-bit result, the 8-bit matrix product, and the
rotation with append to a paged cache.

The reference has none of them (README.md:41-44 of the reference lists the QKV projection, RoPE and the
norm as steps around its kernel that it has not built): **parity unpinned** with respect to the reference.
"""
import torch


def rmsnorm_int8_oracle(x, weight, eps=1e-6, residual=None):
    """x, residual [tokens, hidden] bf16, weight [hidden] bf16.  Returns (t, scale, h): t float64, the
    values in units of the scale BEFORE their rounding to integers (at most half a step from the right
    integer), scale float64 [tokens], and h, the bf16 residual stream."""
    h = x if residual is None else (x.double() + residual.double()).to(torch.bfloat16)
    hw = h.double() * weight.double()
    rstd = (h.double().square().mean(-1) + eps).rsqrt()
    top = hw.abs().amax(-1)
    t = torch.where(top[:, None] > 0, hw * 127.0 / top[:, None].clamp_min(1e-300), torch.zeros_like(hw))
    return t, top * rstd / 127.0, h


def linear_int8_oracle(x, x_scale, weight, weight_scale, bias=None):
    """(out, size): the product in float64, and the sum of the magnitudes of its two terms, which what
    is rounded on the way to it is relative to."""
    y = (x.double() @ weight.double().T) * x_scale.double()[:, None] * weight_scale.double()
    if bias is None:
        return y, y.abs()
    return y + bias.double(), y.abs() + bias.double().abs()


def rope_append_oracle(q, k, v, k_cache, v_cache, page_table, lens, cu_q, inv_freq):
    """Plain loops over the rows (host tensors, lists for the three index arrays; caches
    [num_pages, 128, H_kv, 128]).  Returns (out, k_cache, v_cache, size_q, size_k, dropped): out and
    k_cache float64, out NaN where nothing is written; size_*: |a| + |b| of each rotated pair (0 elsewhere),
    which the rotation's roundings are relative to."""
    num_pages = k_cache.shape[0]
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    kc, vc = k_cache.double().clone(), v_cache.clone()
    size_q, size_k = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(kc.shape, dtype=torch.float64)
    dropped = 0

    def turned(x, pos):
        ang = pos * inv_freq.double()
        c, s = ang.cos(), ang.sin()
        a, b = x[..., :64].double(), x[..., 64:].double()
        size = a.abs() + b.abs()
        return torch.cat([a * c - b * s, b * c + a * s], -1), torch.cat([size, size], -1)

    for i, n in enumerate(lens):
        for t in range(cu_q[i], min(cu_q[i + 1], q.shape[0])):
            pos = n - (cu_q[i + 1] - t)
            if pos < 0:
                dropped += 1
                continue
            out[t], size_q[t] = turned(q[t], pos)
            page = page_table[i][pos // 128] if pos // 128 < len(page_table[i]) else -1
            if not 0 <= page < num_pages:
                dropped += 1
                continue
            kc[page, pos % 128], size_k[page, pos % 128] = turned(k[t], pos)
            vc[page, pos % 128] = v[t]
    return out, kc, vc, size_q, size_k, dropped
