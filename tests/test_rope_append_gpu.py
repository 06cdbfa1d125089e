"""Rotation with append to a paged cache (``ma_rope_append``) against its statement in float64.

Tolerance, from the kernel's arithmetic: the angle is reduced in fp64 and rounded once, half a turn at
most, to 2^-24 of itself: pi 2^-24 radians; sine and cosine are good to 2 ulps (2^-23 at most), two products and
a sum round to 2^-24 each: an output is off by (|a| + |b|) * (pi + 2 + 3) 2^-24, below 9 * 2^-24, and by half a
bf16 step, 2^-8 of its value.  v is copied: equal bits."""
import pytest
import torch

from oracle.int8_oracle import rope_append_oracle
from oracle.producer_oracle import inv_freq_fp32
from megaattention_b200.runtime.rope import default_inv_freq

pytestmark = pytest.mark.gpu


def _close(got, ref, size):
    written = ~ref.isnan()
    tol = size * 9 * 2.0 ** -24 + ref.abs() * 2.0 ** -8 * (1 + 2.0 ** -20)
    d = (got.double() - ref).abs()
    assert bool((d <= tol)[written].all()), float(d[written].max())


def _case(lens_q, lens_k, H, Hkv, seed=0, extra_rows=0, spare=3):
    g = torch.Generator().manual_seed(seed + sum(lens_q) + H)
    t = sum(lens_q) + extra_rows
    c = {"qkv": torch.randn(t, (H + 2 * Hkv) * 128, generator=g).to(torch.bfloat16)}
    need = [-(-n // 128) for n in lens_k]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (max(need) + 1 - n))
        at += n
    c["k_cache"] = torch.randn(pages, 128, Hkv, 128, generator=g).to(torch.bfloat16)
    c["v_cache"] = torch.randn(pages, 128, Hkv, 128, generator=g).to(torch.bfloat16)
    c["table"], c["lens"] = table, list(lens_k)
    c["cu"] = [0]
    for n in lens_q:
        c["cu"].append(c["cu"][-1] + n)
    c["H"], c["Hkv"] = H, Hkv
    return c


def _split(qkv, H, Hkv):
    return [x.unflatten(1, (-1, 128)) for x in qkv.split([H * 128, Hkv * 128, Hkv * 128], dim=1)]


def _run(c, fused=True, out=None, dropped=None, pool=False, inv_freq=None, qkv=None):
    from megaattention_b200.runtime import rope_append
    qkv = c["qkv"].cuda() if qkv is None else qkv
    q, k, v = _split(qkv, c["H"], c["Hkv"])
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    kc, vc = c["k_cache"].cuda(), c["v_cache"].cuda()
    shape = (-1, c["Hkv"], 128) if pool else kc.shape
    i32 = dict(dtype=torch.int32, device="cuda")
    got = rope_append(q, k, v, kc.view(shape), vc.view(shape), torch.tensor(c["table"], **i32),
                      torch.tensor(c["lens"], **i32), torch.tensor(c["cu"], **i32), inv_freq=inv_freq, out=out,
                      dropped=dropped)
    torch.cuda.synchronize()
    return got, kc, vc


def _check(c, got, kc, vc, inv_freq=None):
    q, k, v = _split(c["qkv"], c["H"], c["Hkv"])
    # (the default frequencies as the call makes them: the device's pow, an ulp from the host's here and there)
    w = default_inv_freq(10000.0, "cuda").cpu() if inv_freq is None else inv_freq.cpu()
    out, kr, vr, size_q, size_k, dropped = rope_append_oracle(q, k, v, c["k_cache"], c["v_cache"], c["table"], c["lens"],
                                                              c["cu"], w)
    _close(got.cpu(), out, size_q)
    _close(kc.cpu(), kr, size_k)
    kept = size_k == 0                                   # every other place of the cache: not a bit changed
    assert torch.equal(kc.cpu()[kept], c["k_cache"][kept])
    assert torch.equal(vc.cpu(), vr)
    return dropped


@pytest.mark.parametrize("H,Hkv", [(8, 1), (1, 1), (3, 3), (7, 1), (16, 2), (64, 8)])
@pytest.mark.parametrize("lens_q,lens_k", [([1], [1]), ([1], [129]), ([5, 1, 130], [5, 128, 400]),
                                           ([1] * 40, list(range(1, 41)))])
def test_sizes(lens_q, lens_k, H, Hkv):
    c = _case(lens_q, lens_k, H, Hkv)
    for fused, pool in ((True, False), (False, True)):
        assert _check(c, *_run(c, fused, pool=pool)) == 0


def test_many_sequences_some_of_them_empty():
    lens_q = [0, 0, 3] + [(i * 7) % 4 for i in range(1100)] + [0, 2, 0]
    c = _case(lens_q, [n + (i % 5) for i, n in enumerate(lens_q)], 4, 2)
    assert _check(c, *_run(c)) == 0


def test_far_positions_and_given_frequencies():
    """Angles of 10^5 radians and more: what fp32 products of position and frequency get wrong by 0.004."""
    w = inv_freq_fp32(1e6).cuda()
    c = _case([3, 2], [131072, 70001], 2, 1)
    assert torch.allclose(default_inv_freq(10000.0, "cuda").cpu(), inv_freq_fp32(), rtol=2.0 ** -21, atol=0)
    for inv_freq in (None, w):
        assert _check(c, *_run(c, inv_freq=inv_freq), inv_freq=inv_freq) == 0


def test_rows_behind_the_last_sequence_are_left_alone():
    c = _case([4, 9], [4, 140], 4, 1, extra_rows=6)
    out = torch.full((19, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got, kc, vc = _run(c, out=out)
    assert got is out and bool((out[13:] == 7).all())
    assert _check(c, got, kc, vc) == 0


def test_q_rotated_where_it_is():
    c = _case([4, 9], [4, 140], 4, 2)
    qkv = c["qkv"].cuda()
    q = _split(qkv, 4, 2)[0]
    got, kc, vc = _run(c, out=q, qkv=qkv)
    assert got is q and torch.equal(qkv[:, 512:].cpu(), c["qkv"][:, 512:])
    assert _check(c, got, kc, vc) == 0


def test_rows_without_a_place_are_counted_and_nothing_else_changes():
    """Pages that are not in the cache, a table that is too short, more new rows than keys, no keys at
    all (their bounds checks are tested on the CPU first, tests/test_int8_operators_cpu.py)."""
    c = _case([3, 200, 5, 2, 4], [3, 300, 2, 0, 600], 4, 1)
    c["table"][0][0] = -1
    c["table"][1][1] = 10 ** 6
    c["lens"][4] = 128 * len(c["table"][4]) + 2
    out = torch.full((214, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    dropped = torch.full((1,), 100, dtype=torch.int32, device="cuda")
    got, kc, vc = _run(c, out=out, dropped=dropped)
    want = _check(c, got, kc, vc)
    # 3 of page -1; positions 128-255 of the second (its rows are 100-299); 3 of 5; both; the last two
    assert want == 3 + 128 + 3 + 2 + 2 and int(dropped) == 100 + want
    # rows before their sequence's first key are passed over altogether
    assert bool((out[203:206] == 7).all()) and bool((out[208:210] == 7).all())


def test_no_rows_and_no_sequences():
    c = _case([0, 0], [5, 7], 4, 1, extra_rows=5)
    out = torch.full((5, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got, kc, vc = _run(c, out=out)
    assert bool((out == 7).all()) and torch.equal(kc.cpu(), c["k_cache"]) and torch.equal(vc.cpu(), c["v_cache"])
    c = _case([0, 0], [5, 7], 4, 1)
    assert _run(c)[0].shape == (0, 4, 128)


def test_infinities_and_nan_stay_in_their_rows():
    c = _case([2, 2], [2, 130], 2, 1)
    c["qkv"][1] = float("nan")
    c["qkv"][2, 5] = float("inf")
    got, kc, vc = _run(c)
    out = rope_append_oracle(*_split(c["qkv"], 2, 1), c["k_cache"], c["v_cache"], c["table"], c["lens"], c["cu"],
                             inv_freq_fp32())[0]
    assert torch.equal(got.isnan().cpu() | got.isinf().cpu(), out.isnan() | out.isinf())
    assert torch.equal(vc.cpu().isnan().sum(), torch.tensor(128))       # v of row 1


def test_table_and_lengths_as_views():
    from megaattention_b200.runtime import rope_append
    c = _case([5, 1, 130], [5, 128, 400], 8, 1)
    q, k, v = _split(c["qkv"].cuda(), 8, 1)
    i32 = dict(dtype=torch.int32, device="cuda")
    wide = torch.full((3, 40), -5, **i32)
    n = len(c["table"][0])
    wide[:, 7:7 + n] = torch.tensor(c["table"], **i32)
    kc, vc = c["k_cache"].cuda(), c["v_cache"].cuda()
    got = rope_append(q, k, v, kc, vc, wide[:, 7:7 + n], torch.tensor([0] + c["lens"], **i32)[1:],
                      torch.tensor(c["cu"] + [9], **i32)[:4])
    assert _check(c, got, kc, vc) == 0


def test_a_place_beyond_32_bits_of_elements():
    """Caches of 16500 pages of 8 heads: the last pages start beyond 2^31 elements."""
    from megaattention_b200.runtime import rope_append
    pages = 16500
    kc, vc = (torch.empty(pages, 128, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kc[-3:], vc[-3:] = 1, 1
    c = _case([5, 140], [300, 140], 16, 8, seed=3)
    c["table"] = [[0, 0, pages - 1], [pages - 2, pages - 3, 0]]
    i32 = dict(dtype=torch.int32, device="cuda")
    q, k, v = _split(c["qkv"].cuda(), 16, 8)
    got = rope_append(q, k, v, kc, vc, torch.tensor(c["table"], **i32), torch.tensor(c["lens"], **i32),
                      torch.tensor(c["cu"], **i32))
    c["table"] = [[0, 0, 2], [1, 0, 0]]
    c["k_cache"] = c["v_cache"] = torch.ones(3, 128, 8, 128, dtype=torch.bfloat16)
    assert _check(c, got, kc[-3:], vc[-3:]) == 0


def test_two_rows_with_the_same_place():
    """Either row's key is there in the end, whole, and nothing else changed."""
    c = _case([1, 1], [5, 5], 4, 1)
    c["table"] = [[1, 0], [1, 0]]
    got, kc, vc = _run(c)
    outs = []
    for rows in (0, 1):
        d = dict(c, cu=[0, 1, 1] if rows == 0 else [0, 0, 1], qkv=c["qkv"][rows:rows + 1])
        outs.append(_run(d))
    assert any(torch.equal(kc, o[1]) for o in outs) and any(torch.equal(vc, o[2]) for o in outs)
    assert torch.equal(got, torch.cat([o[0] for o in outs]))


def test_refusals():
    from megaattention_b200.runtime import rope_append
    c = _case([3], [5], 4, 2)
    q, k, v = _split(c["qkv"].cuda(), 4, 2)
    kc, vc = c["k_cache"].cuda(), c["v_cache"].cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, cu = torch.tensor(c["table"], **i32), torch.tensor([5], **i32), torch.tensor([0, 3], **i32)
    ok = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, page_table=table, cache_seqlens=lens, cu_seqlens_q=cu)
    rope_append(**ok)
    for kw in (dict(q=q.float()), dict(k=k[:2]), dict(v=v[:, :1]), dict(q=q[:, :, :64]), dict(q=q.cpu()),
               dict(k_cache=kc[:, :64]), dict(k_cache=kc[:, :, :1]), dict(v_cache=vc[:-1]), dict(page_table=table.long()),
               dict(page_table=table.cpu()), dict(cache_seqlens=torch.cat([lens, lens])), dict(cu_seqlens_q=cu[:1]),
               dict(cu_seqlens_q=[0, 3]), dict(inv_freq=torch.ones(32, device="cuda")), dict(out=q[:, :2]),
               dict(dropped=torch.zeros(1, device="cuda")), dict(page_table=table[:, :0])):
        with pytest.raises((AssertionError, AttributeError)):
            rope_append(**{**ok, **kw})


def test_a_captured_call_follows_the_arrays():
    """A decode step captured once with room for eight rows, replayed as sequences grow and leave."""
    from megaattention_b200.runtime import rope_append
    i32 = dict(dtype=torch.int32, device="cuda")
    c = _case([1] * 8, [120 + i for i in range(8)], 8, 1, spare=20)
    q, k, v = _split(c["qkv"].cuda(), 8, 1)
    kc, vc = c["k_cache"].cuda(), c["v_cache"].cuda()
    table, lens, cu = torch.tensor(c["table"], **i32), torch.tensor(c["lens"], **i32), torch.tensor(c["cu"], **i32)
    w = inv_freq_fp32().cuda()
    out = torch.zeros(8, 8, 128, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rope_append(q, k, v, kc, vc, table, lens, cu, inv_freq=w, out=out)
    for active in (8, 5, 1):
        c["lens"] = [n + 1 for n in c["lens"]]
        c["cu"] = list(range(active + 1)) + [active] * (8 - active)
        c["k_cache"], c["v_cache"] = kc.cpu(), vc.cpu()
        lens.copy_(torch.tensor(c["lens"]))
        cu.copy_(torch.tensor(c["cu"]))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert _check(c, out, kc, vc, w) == 0
        assert bool((out[active:] == 7).all())


def test_an_output_in_another_order_and_one_that_overlaps():
    """Heads before tokens, and rows with room between them; heads that share memory are refused."""
    c = _case([3, 2], [5, 140], 4, 2)
    plain, kc, vc = _run(c)
    for out in (torch.zeros(4, 5, 128, dtype=torch.bfloat16, device="cuda").transpose(0, 1),
                torch.zeros(5, 6, 136, dtype=torch.bfloat16, device="cuda")[:, 1:5, 8:]):
        got, k, v = _run(c, out=out)
        assert got is out and torch.equal(got, plain) and torch.equal(k, kc) and torch.equal(v, vc)
    room = torch.zeros(5 * 4 * 128, dtype=torch.bfloat16, device="cuda")
    for stride in ((128, 128, 1), (384, 128, 1), (512, 64, 1), (128, 512, 1), (0, 128, 1)):
        with pytest.raises(AssertionError):
            _run(c, out=room.as_strided((5, 4, 128), stride))
    one = dict(c, cu=[0, 1, 1], lens=[5, 0], qkv=c["qkv"][:1])              # (a single token: any step between tokens)
    got, _, _ = _run(one, out=room.as_strided((1, 4, 128), (0, 128, 1)))
    assert torch.equal(got, _run(one)[0])


def test_an_output_that_shares_memory_with_the_inputs():
    """Another token's or head's memory is refused (it would be read before or after it is written); q itself and
    what lies between the inputs' tokens or heads is not."""
    c = _case([3, 60], [5, 140], 4, 2)
    want, kc, vc = _run(c)
    t, n = 63, (4 + 2 * 2) * 128
    i32 = dict(dtype=torch.int32, device="cuda")
    index = [torch.tensor(c[x], **i32) for x in ("table", "lens", "cu")]

    def run(q, k, v, out):
        from megaattention_b200.runtime import rope_append
        k2, v2 = c["k_cache"].cuda(), c["v_cache"].cuda()
        return rope_append(q, k, v, k2, v2, *index, out=out), k2, v2

    room = torch.zeros(3 * t * n, dtype=torch.bfloat16, device="cuda")
    qkv = room[t * n:2 * t * n].view(t, n)
    qkv.copy_(c["qkv"])
    q, k, v = _split(qkv, 4, 2)
    before = room.clone()
    for shift, stride in ((0, (512, 128)), (n, (n, 128)), (-n, (n, 128)), (8, (n, 128)), (-128, (n, 128)), (128, (n, 128)),
                          (512, (n, 128)), (768, (n, 128)), (0, (n, 256)), (0, (128, t * 128)), (t * n - 128, (512, 128)),
                          (-512 * t + 128, (512, 128)), (-512, (n, 128))):
        with pytest.raises(AssertionError):
            run(q, k, v, room.as_strided((t, 4, 128), (*stride, 1), t * n + shift))
    assert torch.equal(room, before)
    # a place of its own between the tokens, before q and behind v; between the heads; behind everything
    wide = torch.zeros(t, n + 1024 + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, 512:512 + n] = qkv
    pairs = torch.zeros(t, 4, 2, 128, dtype=torch.bfloat16, device="cuda")
    pairs[:, :, 0] = q
    packed = (q.contiguous(), k.contiguous(), v.contiguous())
    for ins, out in ((_split(wide[:, 512:512 + n], 4, 2), wide[:, :512].unflatten(1, (4, 128))),
                     (_split(wide[:, 512:512 + n], 4, 2), wide[:, 512 + n:1024 + n].unflatten(1, (4, 128))),
                     ((pairs[:, :, 0], k, v), pairs[:, :, 1]), (packed, pairs[:, :, 1]),
                     ((q, k, v), room[2 * t * n:][:512 * t].view(t, 4, 128)), ((q, k, v), q)):
        got, k2, v2 = run(*ins, out)
        assert got is out and torch.equal(got, want) and torch.equal(k2, kc) and torch.equal(v2, vc)
    one = [x[:1] for x in _split(c["qkv"].cuda(), 4, 2)]
    index = [torch.tensor(x, **i32) for x in (c["table"], [5, 0], [0, 1, 1])]
    with pytest.raises(AssertionError):                  # a single token: k's heads are k's all the same
        run(*one, one[0].as_strided((1, 4, 128), (8, 128, 1), 128))
    first = run(*one, None)[0]
    assert torch.equal(run(*one, one[0].as_strided((1, 4, 128), (8, 128, 1)))[0], first)


@pytest.mark.parametrize("batch", [2, 30, 31, 32, 33, 64])
@pytest.mark.parametrize("empty", [(), (0,), (-1,), (0, 1, -2, -1), "odd", "even"])
def test_batches_around_a_warp_with_empty_sequences(batch, empty):
    """Up to 31 sequences are looked through at once, more in rounds; the first and the last of them empty or not."""
    gone = {b for b in range(batch) if b % 2 == (empty == "odd")} if isinstance(empty, str) else {e % batch for e in empty}
    lens_q = [0 if b in gone else 1 + b % 3 for b in range(batch)]
    c = _case(lens_q, [n + 100 + 9 * b for b, n in enumerate(lens_q)], 4, 2)
    if not sum(lens_q):
        assert _run(c)[0].shape[0] == 0
        return
    assert _check(c, *_run(c)) == 0
