"""The operators between two layers in the order a serving step runs them: norm to 8 bits, 8-bit QKV
projection, rotation and append to the paged cache, the paged layer, norm of its output to 8 bits, the
next projection - on one stream with no host synchronisation of the operators' own, against float64
arithmetic on what each stage was given."""
import pytest
import torch

from oracle.chain_oracle import err_beyond_rounding, full_chain_oracle
from oracle.int8_oracle import linear_int8_oracle, rmsnorm_int8_oracle, rope_append_oracle
from oracle.producer_oracle import inv_freq_fp32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens_q,lens_k,H,Hkv,hidden", [
    ([150, 260], [150, 516], 4, 2, 512),
    ([1, 1, 1], [130, 1, 300], 8, 1, 1000),              # a decode step
    ([64, 200, 256], [64, 200, 256], 8, 1, 1024),
])
def test_a_whole_layer_step_in_eight_bits(lens_q, lens_k, H, Hkv, hidden):
    from megaattention_b200.runtime import (
        FusedFaOprojArWorkspace, FusedPrefillLayer, check_linear_status, linear_int8, quantize_weight_int8,
        residual_rmsnorm_int8, rmsnorm_int8, rope_append)
    g = torch.Generator().manual_seed(sum(lens_k) + hidden)

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16)

    t, width = sum(lens_q), (H + 2 * Hkv) * 128
    x, wn1, wn2 = randn(t, hidden), 1 + randn(hidden, std=0.1), 1 + randn(hidden, std=0.1)
    W_qkv, W_up, W_o = randn(width, hidden, std=hidden ** -0.5), randn(640, hidden, std=hidden ** -0.5), randn(
        H * 128, hidden, std=(H * 128) ** -0.5)
    need = [-(-n // 128) for n in lens_k]
    pages = sum(need) + 2
    order, table, at = torch.randperm(pages, generator=g).tolist(), [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (max(need) - n))
        at += n
    kc, vc = randn(pages, 128, Hkv, 128), randn(pages, 128, Hkv, 128)
    cu = [0]
    for n in lens_q:
        cu.append(cu[-1] + n)

    i32 = dict(dtype=torch.int32, device="cuda")
    xd, kcd, vcd = x.cuda(), kc.cuda(), vc.cuda()
    qkv8, up8 = quantize_weight_int8(W_qkv.cuda()), quantize_weight_int8(W_up.cuda())
    table_d, lens_d, cu_d = torch.tensor(table, **i32), torch.tensor(lens_k, **i32), torch.tensor(cu, **i32)
    dropped = torch.zeros(1, **i32)
    tiles = sum(-(-n // 128) for n in lens_q)
    ws = FusedFaOprojArWorkspace.create(None, tiles, hidden, H, 128, q_per_kv=H // Hkv, device="cuda:0", paged=True,
                                        max_num_batch=len(lens_q), max_num_pages=pages,
                                        max_num_pages_per_seq=max(need))
    ws.compile()
    layer = FusedPrefillLayer(ws, W_o.cuda() if hidden % 64 == 0 else W_o)
    w = inv_freq_fp32().cuda()
    n1, s1 = rmsnorm_int8(xd, wn1.cuda())
    qkv = linear_int8(n1, s1, *qkv8)
    q, k, v = (p.unflatten(1, (-1, 128)) for p in qkv.split([H * 128, Hkv * 128, Hkv * 128], dim=1))
    q = rope_append(q, k, v, kcd, vcd, table_d, lens_d, cu_d, inv_freq=w, dropped=dropped)
    layer(q, kcd, vcd, torch.tensor(cu), page_table=table_d, cache_seqlens=lens_d)
    n2, s2, res = residual_rmsnorm_int8(ws, xd.clone(), wn2.cuda(), inplace=True)
    up = linear_int8(n2, s2, *up8)
    ws.check_status()
    check_linear_status()
    assert int(dropped) == 0

    # each stage on what it was given
    tt, ss, _ = rmsnorm_int8_oracle(x, wn1)
    assert bool(((n1.cpu().double() - tt).abs() <= 0.5 + 127 * 2.0 ** -23).all())
    ref, size = linear_int8_oracle(n1.cpu(), s1.cpu(), *(p.cpu() for p in qkv8))
    assert bool(((qkv.cpu().double() - ref).abs() <= 2.0 ** -8 * 1.001 * size).all())
    qh, kh, vh = (p.unflatten(1, (-1, 128)) for p in qkv.cpu().split([H * 128, Hkv * 128, Hkv * 128], dim=1))
    out, kr, vr, size_q, size_k, _ = rope_append_oracle(qh, kh, vh, kc, vc, table, lens_k, cu, w.cpu())
    assert bool(((q.cpu().double() - out).abs() <= size_q * 9 * 2.0 ** -24 + out.abs() * 2.0 ** -8 * 1.001).all())
    assert bool(((kcd.cpu().double() - kr).abs() <= size_k * 9 * 2.0 ** -24 + kr.abs() * 2.0 ** -8 * 1.001).all())
    assert torch.equal(vcd.cpu(), vr)
    # the layer reads from the pages what was appended
    ks = torch.cat([kcd.cpu()[table[b][:need[b]]].reshape(-1, Hkv, 128)[:n] for b, n in enumerate(lens_k)])
    vs = torch.cat([vcd.cpu()[table[b][:need[b]]].reshape(-1, Hkv, 128)[:n] for b, n in enumerate(lens_k)])
    _, yp, _ = full_chain_oracle(q.cpu(), ks, vs, W_o, lens_q, lens_k)
    y = layer.output().cpu()
    assert err_beyond_rounding(y, yp) <= 8e-3            # the layer's own tolerance with cached keys
    tt, ss, h = rmsnorm_int8_oracle(y, wn2, 1e-6, x)
    assert torch.equal(res.cpu(), h) and bool(((n2.cpu().double() - tt).abs() <= 0.5 + 127 * 2.0 ** -23).all())
    ref, size = linear_int8_oracle(n2.cpu(), s2.cpu(), *(p.cpu() for p in up8))
    assert bool(((up.cpu().double() - ref).abs() <= 2.0 ** -8 * 1.001 * size).all())


def _operators():
    """Each operator, small, as a call without arguments and the number of outputs that it allocates."""
    from megaattention_b200.runtime import dequantize_int8, linear_int8, rmsnorm_int8, rope_append
    from megaattention_b200.runtime.rope import default_inv_freq
    x, w = torch.ones(5, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q8, s8 = torch.ones(5, 64, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda")
    h = torch.ones(5, 2, 128, dtype=torch.bfloat16, device="cuda")
    pages = torch.zeros(1, 128, 2, 128, dtype=torch.bfloat16, device="cuda")
    i = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0]], [3], [0, 3])]
    freq = default_inv_freq(1e4, "cuda")
    return [(lambda: rmsnorm_int8(x, w, residual=x), 3), (lambda: linear_int8(q8, s8, q8, s8), 1),
            (lambda: dequantize_int8(q8, s8), 1), (lambda: rope_append(h, h, h, pages, pages, *i, inv_freq=freq), 1)]


def test_a_dispatch_mode_sees_the_outputs():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(str(func))
            return func(*args, **(kwargs or {}))

    for call, outputs in _operators():
        want, names = call(), []
        with Seen():
            got = call()
        assert sum("aten.empty" in n for n in names) == outputs, names
        for a, b in zip(want if outputs > 1 else [want], got if outputs > 1 else [got]):
            assert torch.equal(a[:3], b[:3])             # (the append's last rows are behind its sequence)


def test_fresh_outputs_are_filled_where_torch_fills_them():
    """Rows that the append does not write: NaN under deterministic algorithms, not what the memory held."""
    call = _operators()[-1][0]
    torch.use_deterministic_algorithms(True)
    try:
        for _ in range(3):
            old = torch.full((5, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda")
            del old                                      # (its memory is the next of this size)
            out = call()
            assert bool(out[3:].isnan().all()) and bool(out[:3].isfinite().all())
            del out
    finally:
        torch.use_deterministic_algorithms(False)
