"""Residual add + RMSNorm with an 8-bit result (``ma_rmsnorm_quant``) against its statement in
float64.

Tolerances, from the kernel's arithmetic.  An integer is the rounding of h w (exact in fp32) times 127 /
max|h w|: one division and one product, each off by 2^-24 of at most 127, so that it lies within half a step
and 127 * 2^-23 of the exact value.  A scale is max * rsqrt(sum / n + eps) / 127: the sum of squares is a
chain of at most 32 fused steps per thread, 5 between lanes and 16 between warps, each off by half an
ulp, of which the root takes half: 27 * 2^-24; the root itself 2 ulps (4 * 2^-24), five more products
and sums 5 * 2^-24: below 40 * 2^-24.  The residual stream is one rounding, the same one: equal bits."""
import pytest
import torch

from oracle.int8_oracle import rmsnorm_int8_oracle

pytestmark = pytest.mark.gpu
STEP = 0.5 + 127 * 2.0 ** -23
SCALE = 40 * 2.0 ** -24


def _check(q, scale, x, w, eps, residual=None, new=None):
    t, s, h = rmsnorm_int8_oracle(x.cpu(), w.cpu(), eps, None if residual is None else residual.cpu())
    assert q.dtype == torch.int8 and q.shape == x.shape and scale.dtype == torch.float32
    assert bool(((q.cpu().double() - t).abs() <= STEP).all())
    assert bool(((scale.cpu().double() - s).abs() <= s * SCALE).all())
    if residual is not None:
        assert torch.equal(new.cpu(), h)


def _inputs(tokens, hidden, seed=0):
    g = torch.Generator().manual_seed(tokens * 31 + hidden + seed)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16)
    r = (3 * torch.randn(tokens, hidden, generator=g)).to(torch.bfloat16)
    w = (1 + 0.3 * torch.randn(hidden, generator=g)).to(torch.bfloat16)
    return x.cuda(), r.cuda(), w.cuda()


@pytest.mark.parametrize("hidden", [8, 72, 256, 1000, 1024, 1032, 2048, 2056, 4096, 5480, 8192, 8200, 16384])
@pytest.mark.parametrize("tokens", [1, 7, 1300])
def test_packed_rows(tokens, hidden):
    from megaattention_b200.runtime import rmsnorm_int8
    x, r, w = _inputs(tokens, hidden)
    q, scale = rmsnorm_int8(x, w, 1e-5)
    _check(q, scale, x, w, 1e-5)
    assert q.stride(0) % 16 == 0 or tokens == 1
    r0 = r.clone()
    q, scale, new = rmsnorm_int8(x, w, 1e-6, residual=r)
    assert torch.equal(r, r0) and new.data_ptr() != r.data_ptr()       # not in place unless asked
    _check(q, scale, x, w, 1e-6, r0, new)
    q2, scale2, same = rmsnorm_int8(x, w, 1e-6, residual=r, inplace=True)
    assert same is r and torch.equal(q, q2) and torch.equal(scale, scale2) and torch.equal(new, r)


def test_rows_beyond_32_bits_of_elements():
    from megaattention_b200.runtime import dequantize_int8, rmsnorm_int8
    tokens, hidden = 135000, 16384
    x = torch.empty(tokens, hidden, dtype=torch.bfloat16, device="cuda")
    rows, r, w = _inputs(7, hidden)
    at = torch.tensor([0, 1, 65535, 131071, 131072, tokens - 2, tokens - 1], device="cuda")
    x[at] = rows
    q, scale = rmsnorm_int8(x, w)
    _check(q[at], scale[at], rows, w, 1e-6)
    for a in at.tolist():
        x[a] = float("nan")
    out = dequantize_int8(q, scale, out=x)
    assert torch.equal(out[at], (q[at].float() * scale[at, None]).bfloat16())


def test_no_rows():
    from megaattention_b200.runtime import rmsnorm_int8
    x, r, w = _inputs(0, 64)
    q, scale = rmsnorm_int8(x, w)
    assert q.shape == (0, 64) and scale.shape == (0,)
    assert rmsnorm_int8(x, w, residual=r)[2].shape == (0, 64)


def test_rows_with_pitches_and_outputs_given():
    """Views of wider tensors on every side: what is between the rows stays as it is."""
    from megaattention_b200.runtime import rmsnorm_int8
    tokens, hidden = 37, 1000
    x, r, w = _inputs(tokens, hidden)
    wide = lambda t, pad, dtype=torch.bfloat16: torch.full((tokens, hidden + pad), 5, dtype=dtype, device="cuda")  # noqa: E731
    xs, rs, qs = wide(x, 24), wide(r, 8), wide(x, 24, torch.int8)
    xs[:, 8:8 + hidden], rs[:, :hidden] = x, r
    scale = torch.empty(tokens, device="cuda")
    q, s, new = rmsnorm_int8(xs[:, 8:8 + hidden], w, residual=rs[:, :hidden], inplace=True, out=qs[:, 0:hidden],
                             scale=scale)
    assert s is scale and q.data_ptr() == qs.data_ptr()
    _check(qs[:, :hidden], scale, x, w, 1e-6, r, rs[:, :hidden])
    assert bool((qs[:, hidden:] == 5).all()) and bool((rs[:, hidden:] == 5).all())


@pytest.mark.parametrize("hidden", [64, 2048, 16384])
def test_rows_of_zeros_tiny_rows_and_rows_that_are_not_finite(hidden):
    from megaattention_b200.runtime import rmsnorm_int8
    x, _, w = _inputs(9, hidden)
    x[1] = 0
    x[2, hidden // 2] = float("nan")
    x[3, hidden - 1] = float("inf")
    x[4, 0] = float("-inf")
    x[5] = 3e38                                       # the sum of squares overflows
    x[6] = 1e-38                                      # below every scale in use
    x[7] = 1e-30
    for eps in (1e-6, 0.0):
        q, scale = rmsnorm_int8(x, w, eps)
        q, scale = q.cpu(), scale.cpu()
        for row in (2, 3, 4, 5):
            assert bool(scale[row].isnan()) and int(q[row].abs().max()) == 0
        for row in (1, 6):
            assert float(scale[row]) == 0 and int(q[row].abs().max()) == 0
        keep = [0, 8] if eps == 0 else [0, 7, 8]
        _check(q[keep], scale[keep], x[keep], w, eps)
        if eps == 0:                                  # 1e-60 is no fp32 number: 1 / 0
            assert bool(scale[7].isnan()) and int(q[7].abs().max()) == 0
    w[0] = float("nan")
    assert bool(rmsnorm_int8(x, w)[1].isnan().all())


@pytest.mark.parametrize("hidden", [64, 1000, 2048, 16384])
@pytest.mark.parametrize("residual", [False, True])
def test_rows_whose_squares_fp32_does_not_hold(hidden, residual):
    """Rows of 2^-k: right down to a mean of 2^-126, where n squares off by 2^-150 at most are 2^-24 of it (the
    tolerance has that, as a rounding more); NaN below, not a scale from squares of a few bits; right again
    behind an eps that is larger."""
    from megaattention_b200.runtime import rmsnorm_int8
    powers = [0, 50, 60, 62, 64, 65, 66, 68, 70, 73, 80, 100, 110]
    x, r, w = _inputs(len(powers), hidden)
    down = torch.tensor([2.0 ** -k for k in powers], device="cuda")[:, None]
    x = (x.float() * down).bfloat16()                  # (exact)
    r = (r.float() * down).bfloat16() if residual else None
    h = x.double() + r.double() if residual else x.double()
    mean = h.square().mean(-1).cpu()
    for eps in (0.0, 2.0 ** -140, 2.0 ** -100, 1e-6):
        got = rmsnorm_int8(x, w, eps, residual=r)
        q, scale = got[0].cpu(), got[1].cpu()
        keep = [i for i in range(len(powers)) if float(mean[i]) + eps >= 2.0 ** -125.9]
        lost = [i for i in range(len(powers)) if float(mean[i]) + eps < 2.0 ** -126.1]
        assert len(keep) + len(lost) == len(powers) and len(lost) in ((0,) if eps > 2.0 ** -120 else range(7, 11))
        _check(q[keep], scale[keep], x[keep], w, eps, None if r is None else r[keep], got[2][keep] if residual else None)
        assert bool(scale[lost].isnan().all()) and not bool(q[lost].any())


def test_tiles_of_the_fused_output_in_place():
    """Three ragged sequences in csym; padding rows hold NaN and are not read as tokens."""
    from megaattention_b200.metadata import build_row_desc
    from megaattention_b200.runtime import FusedFaOprojArWorkspace, residual_rmsnorm, residual_rmsnorm_int8
    for hidden in (1000, 4096):
        sq = [300, 129, 64]
        meta = build_row_desc(sq)
        ws = FusedFaOprojArWorkspace.create(None, meta.num_row_tiles, hidden, 2, 128, q_per_kv=2,
                                            max_tot_k=sum(sq), device="cuda:0")
        ws.compile()
        ws.set_meta(meta)
        y, r, w = _inputs(sum(sq), hidden)
        tiles = torch.full((meta.num_row_tiles, 128, ws.num_out * 128), float("nan"), device="cuda", dtype=torch.bfloat16)
        a = t = 0
        for n in sq:
            for i in range(0, n, 128):
                tiles[t, :min(128, n - i), :hidden] = y[a + i:a + min(n, i + 128)]
                t += 1
            a += n
        ws.csym.copy_(tiles.view(ws.csym.shape))
        q, scale, new = residual_rmsnorm_int8(ws, r, w, 1e-5)
        _check(q, scale, y, w, 1e-5, r, new)
        normed, same = residual_rmsnorm(ws, r, w, 1e-5, inplace=True)      # the bf16 form's stream
        assert torch.equal(same, new)
        q2, _, _ = residual_rmsnorm_int8(ws, r, w, 1e-5, inplace=True, out=q, meta=meta)
        assert q2 is q


def test_the_fused_output_from_another_stream():
    """Runs on the workspace's stream, results allocated there, whatever stream is current."""
    from megaattention_b200.metadata import build_row_desc
    from megaattention_b200.runtime import FusedFaOprojArWorkspace, residual_rmsnorm_int8
    meta = build_row_desc([128])
    ws = FusedFaOprojArWorkspace.create(None, 1, 512, 2, 128, q_per_kv=2, max_tot_k=128, device="cuda:0")
    ws.compile()
    ws.set_meta(meta)
    y, r, w = _inputs(128, 512)
    ws.csym.copy_(y.view(ws.csym.shape))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q, scale, new = residual_rmsnorm_int8(ws, r, w, 1e-5)
        assert torch.cuda.current_stream() == side
    ws._stream().synchronize()
    _check(q, scale, y, w, 1e-5, r, new)
    with pytest.raises(AssertionError):
        residual_rmsnorm_int8(ws, r[:100], w)
    with pytest.raises(AssertionError):
        residual_rmsnorm_int8(ws, None, w)


def test_refusals():
    from megaattention_b200.runtime import rmsnorm_int8
    x, r, w = _inputs(4, 64)
    for bad in (lambda: rmsnorm_int8(x.float(), w), lambda: rmsnorm_int8(x, w[:32]), lambda: rmsnorm_int8(x.cpu(), w),
                lambda: rmsnorm_int8(x[:, :60], w[:60]), lambda: rmsnorm_int8(x.T, w), lambda: rmsnorm_int8(x, w.float()),
                lambda: rmsnorm_int8(x, w, residual=r[:3]), lambda: rmsnorm_int8(x, w, inplace=True),
                lambda: rmsnorm_int8(x, w, residual=r.cpu()), lambda: rmsnorm_int8(x[:, 1:57], w[1:57]),
                lambda: rmsnorm_int8(x, w, out=torch.empty(4, 64, device="cuda")),
                lambda: rmsnorm_int8(x, w, scale=torch.empty(3, device="cuda")),
                lambda: rmsnorm_int8(x[None], w)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(RuntimeError):
        rmsnorm_int8(x, w, -1.0)


def test_captured_call_and_another_stream():
    from megaattention_b200.runtime import rmsnorm_int8
    x, r, w = _inputs(33, 4096)
    want = rmsnorm_int8(x, w, residual=r)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = rmsnorm_int8(x, w, residual=r)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rmsnorm_int8(x, w, residual=r)
    x2, r2, _ = _inputs(33, 4096, seed=1)
    x.copy_(x2)
    r.copy_(r2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(rmsnorm_int8(x2, w, residual=r2), out))


@pytest.mark.parametrize("tokens,hidden", [(700, 512), (700, 4096), (37, 16384), (1, 1024)])
def test_outputs_that_share_memory(tokens, hidden):
    """What another row reads, or two outputs write, is refused; integers in their own row of x, column slices of one
    buffer and a residual that is x itself are not, and are right."""
    from megaattention_b200.runtime import rmsnorm_int8
    x, r, w = _inputs(tokens, hidden)
    want, want_r = rmsnorm_int8(x, w), rmsnorm_int8(x, w, residual=r)

    def half(t, second=False):                             # of each row's bytes: where its integers find room
        return t.view(torch.int8)[:, hidden:] if second else t.view(torch.int8)[:, :hidden]

    for second in (False, True):
        own, other = x.clone(), r.clone()
        got = rmsnorm_int8(own, w, out=half(own, second))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got = rmsnorm_int8(x, w, residual=other, out=half(other, second))
        assert all(torch.equal(a, b) for a, b in zip(got, want_r))
    both = torch.cat([x, r], 1)
    got = rmsnorm_int8(both[:, :hidden], w, residual=both[:, hidden:], inplace=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want_r)) and torch.equal(both[:, :hidden], x)
    twice = x.clone()
    got = rmsnorm_int8(twice, w, residual=twice, inplace=True)
    _check(got[0], got[1], x, w, 1e-6, x, got[2])

    room = torch.zeros(tokens + 2, hidden, dtype=torch.bfloat16, device="cuda")
    mid = room[1:-1]
    mid.copy_(x)
    before, floats = room.clone(), room.view(-1).view(torch.float32)
    eight = torch.zeros(tokens, hidden, dtype=torch.int8, device="cuda")
    bad = [dict(scale=floats[hidden // 2:][:tokens]), dict(out=half(mid), residual=mid, inplace=True),
           dict(out=eight, scale=eight.view(-1).view(torch.float32)[:tokens])]
    if tokens > 1:                                         # other rows' memory
        bad += [dict(out=mid.view(torch.int8).view(-1)[:tokens * hidden].view(tokens, hidden)), dict(out=half(room[:-2])),
                dict(out=half(room[2:], True)), dict(residual=room[:-2], inplace=True), dict(residual=room[2:], inplace=True)]
    for kw in bad:
        with pytest.raises(AssertionError):
            rmsnorm_int8(mid, w, **kw)
    with pytest.raises(AssertionError):
        rmsnorm_int8(mid[:1], mid[0], out=half(mid[:1]))   # its own weights
    assert torch.equal(room, before)
