"""Matrix product of 8-bit integers (``ma_linear_quant``) against float64.

Tolerance, from the kernel's arithmetic: the sum is exact; its conversion to fp32, two products with the
scales and the sum with the bias are off by 2^-24 of the product's (and the bias's) magnitude each, the
result's own rounding by half a step: 2^-8 (bf16) or 2^-24 (fp32) of the value.  Values that are exact
in between have to be exact at the end (``test_sums_are_exact``)."""
import pytest
import torch

from oracle.int8_oracle import linear_int8_oracle

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _rows(rows, cols, g, pitch=None):
    """int8 rows, 16 bytes apart or `pitch`; what is between them is 99, and has no part in the sums."""
    pitch = pitch or -(-cols // 16) * 16
    t = torch.full((rows, pitch), 99, dtype=torch.int8)
    t[:, :cols] = torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int8)
    return t.cuda()[:, :cols]


def _case(m, k, n, bias, seed=0):
    g = torch.Generator().manual_seed(m * 7 + k * 3 + n + seed)
    x, w = _rows(m, k, g), _rows(n, k, g)
    xs, ws = torch.rand(m, generator=g) + 0.01, (torch.rand(n, generator=g) + 0.01) / (k ** 0.5 * 64)
    b = torch.randn(n, generator=g).to(torch.bfloat16).cuda() if bias else None
    return x, xs.cuda(), w, ws.cuda(), b


def _check(out, x, xs, w, ws, b):
    ref, size = linear_int8_oracle(x, xs, w, ws, b)
    assert out.shape == ref.shape
    tol = 4 * 2.0 ** -24 * size + HALF[out.dtype] * ref.abs() * (1 + 2.0 ** -20)
    bad = (out.double() - ref).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 255, 300])
@pytest.mark.parametrize("k,n", [(1, 1), (16, 8), (100, 130), (127, 128), (1000, 1001), (4096, 384)])
def test_sizes(m, k, n):
    from megaattention_b200.runtime import check_linear_status, linear_int8
    x, xs, w, ws, b = _case(m, k, n, (m + n) % 2 == 0)
    for dtype in (torch.bfloat16, torch.float32):
        _check(linear_int8(x, xs, w, ws, bias=b, out_dtype=dtype), x, xs, w, ws, b)
    check_linear_status()


@pytest.mark.parametrize("m,k,n", [(1, 16384, 2304), (48, 4096, 10240), (513, 640, 2304), (1384, 4096, 1280),
                                   (2049, 1152, 4104), (4100, 200, 1000), (1000, 4096, 16384)])
@pytest.mark.parametrize("bias", [False, True])
def test_large_sizes(m, k, n, bias):
    from megaattention_b200.runtime import check_linear_status, linear_int8
    x, xs, w, ws, b = _case(m, k, n, bias)
    _check(linear_int8(x, xs, w, ws, bias=b), x, xs, w, ws, b)
    check_linear_status()


@pytest.mark.parametrize("m,k,n", [(3, 131071, 40), (300, 131071, 200), (600, 131071, 200)])
def test_the_longest_sums_are_exact(m, k, n):
    """-128 throughout: 131071 * 2^14 is the largest sum that can come up, just below 2^31."""
    from megaattention_b200.runtime import linear_int8
    pad = torch.full((max(m, n), 131072), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(max(m, n), device="cuda")
    out = linear_int8(pad[:m, :k], one[:m], pad[:n, :k], one[:n], out_dtype=torch.float32)
    assert bool((out == float(torch.tensor(float(k * 2 ** 14), dtype=torch.float32))).all())
    with pytest.raises(RuntimeError):                 # one more could pass 32 bits
        linear_int8(pad[:m], one[:m], pad[:n], one[:n])


def test_sums_are_exact():
    """Small integers with scales of one: every output is a whole number below 2^24."""
    from megaattention_b200.runtime import linear_int8
    for m in (5, 40, 200, 700):
        g = torch.Generator().manual_seed(m)
        x, w = _rows(m, 700, g), _rows(333, 700, g)
        one = torch.ones(max(m, 333), device="cuda")
        out = linear_int8(x, one[:m], w, one[:333], out_dtype=torch.float32)
        assert torch.equal(out.double(), x.double() @ w.double().T)


@pytest.mark.parametrize("m", [9, 100, 600])
def test_pitches_and_a_given_output(m):
    from megaattention_b200.runtime import linear_int8
    g = torch.Generator().manual_seed(m)
    x, w = _rows(m, 333, g, 352), _rows(300, 333, g, 1008)
    xs, ws = torch.rand(m, generator=g).cuda(), torch.rand(300, generator=g).cuda() / 1000
    for dtype in (torch.bfloat16, torch.float32):
        for pitch, at in ((301, 0), (304, 0), (400, 3), (512, 64)):       # odd rows, whole rows, odd start
            buf = torch.full((m + 1, pitch), -7.0, dtype=dtype, device="cuda")
            out = buf[:m, at:at + 300]
            assert linear_int8(x, xs, w, ws, out=out) is out
            _check(out, x, xs, w, ws, None)
            rest = buf.clone()
            rest[:m, at:at + 300] = -7.0
            assert bool((rest == -7.0).all())


@pytest.mark.parametrize("m,n", [(70000, 32768), (3, 500000)])
def test_outputs_beyond_32_bits_of_elements_and_wide_ones(m, n):
    from megaattention_b200.runtime import check_linear_status, linear_int8
    g = torch.Generator().manual_seed(m)
    x, w = _rows(m, 48, g), _rows(n, 48, g)
    xs, ws = torch.rand(m, generator=g).cuda(), torch.rand(n, generator=g).cuda() / 1000
    out = linear_int8(x, xs, w, ws)
    at = torch.tensor(sorted({0, 1, m // 2, m - 2, m - 1}), device="cuda")
    _check(out[at], x[at], xs[at], w, ws, None)
    check_linear_status()


def test_nothing_to_do_and_scales_that_are_not_finite():
    from megaattention_b200.runtime import linear_int8
    x, xs, w, ws, b = _case(20, 64, 48, True)
    assert linear_int8(x[:0], xs[:0], w, ws, bias=b).shape == (0, 48)
    assert linear_int8(x, xs, w[:0], ws[:0]).shape == (20, 0)
    xs[3] = float("nan")
    ws[5] = float("inf")
    out = linear_int8(x, xs, w, ws, bias=b).float()
    assert bool(out[3].isnan().all())
    col = out[:, 5]
    assert not bool(col.isfinite().any())
    keep = torch.ones(20, dtype=torch.bool, device="cuda")
    keep[3] = False
    cols = torch.ones(48, dtype=torch.bool, device="cuda")
    cols[5] = False
    _check(out[keep][:, cols].bfloat16(), x[keep].contiguous(), xs[keep], w[cols].contiguous(), ws[cols], b[cols])


def test_refusals():
    from megaattention_b200.runtime import linear_int8
    x, xs, w, ws, b = _case(20, 64, 48, True)
    for bad in (lambda: linear_int8(x.float(), xs, w, ws), lambda: linear_int8(x, xs[:5], w, ws),
                lambda: linear_int8(x, xs, w[:, :48], ws), lambda: linear_int8(x, xs, w, ws, bias=b.float()),
                lambda: linear_int8(x, xs, w, ws, out_dtype=torch.float16), lambda: linear_int8(x.cpu(), xs, w, ws),
                lambda: linear_int8(x[:, :50].contiguous(), xs, w[:, :50].contiguous(), ws),
                lambda: linear_int8(x, xs, w, ws, out=torch.empty(20, 47, device="cuda")),
                lambda: linear_int8(x, xs, w, ws, out=torch.empty(1, 48, device="cuda").expand(20, 48)),
                lambda: linear_int8(x, xs.bfloat16(), w, ws), lambda: linear_int8(x[:, 1:], xs, w[:, 1:], ws),
                lambda: linear_int8(x, xs, w, ws, out=torch.empty(48, 20, device="cuda").T)):
        with pytest.raises(AssertionError):
            bad()


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 16), (70, 1000), (5, 1001), (2000, 4096), (40000, 24)])
def test_eight_bits_as_the_values_they_stand_for(rows, cols):
    """One product in fp32 and one rounding: equal bits."""
    from megaattention_b200.runtime import dequantize_int8
    g = torch.Generator().manual_seed(rows + cols)
    q, s = _rows(rows, cols, g), torch.rand(rows, generator=g).cuda()
    q[0, 0] = -128
    for dtype in (torch.bfloat16, torch.float32):
        want = (q.float() * s[:, None]).to(dtype)
        assert torch.equal(dequantize_int8(q, s, out_dtype=dtype), want)
        buf = torch.full((rows, cols + 5), -7.0, dtype=dtype, device="cuda")
        assert torch.equal(dequantize_int8(q, s, out=buf[:, 3:3 + cols]), want)
        assert bool((buf[:, :3] == -7).all()) and bool((buf[:, 3 + cols:] == -7).all())
    assert dequantize_int8(q[:0], s[:0]).shape == (0, cols)
    with pytest.raises(AssertionError):
        dequantize_int8(q.float(), s)


@pytest.mark.parametrize("tokens", [8, 700])
def test_weights_written_by_the_kernel_before(tokens):
    """The projection starts while the kernel before it ends, and sends for its first weights then: a weight
    that this very kernel writes is the new one all the same, every time."""
    from megaattention_b200.runtime import linear_int8, rmsnorm_int8
    g = torch.Generator().manual_seed(tokens)
    x, xs = _rows(tokens, 2048, g), torch.rand(tokens, generator=g).cuda()
    ones = torch.ones(2048, dtype=torch.bfloat16, device="cuda")
    keys = [torch.randn(3000, 2048, generator=g).bfloat16().cuda() for _ in range(4)]
    want = [linear_int8(x, xs, *rmsnorm_int8(k, ones)) for k in keys]
    torch.cuda.synchronize()
    w, ws = torch.empty(3000, 2048, dtype=torch.int8, device="cuda"), torch.empty(3000, device="cuda")
    outs = []
    for i in range(40):
        rmsnorm_int8(keys[i % 4], ones, out=w, scale=ws)
        outs.append(linear_int8(x, xs, w, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 4]) for i, o in enumerate(outs))


def test_captured_calls_two_streams_and_equal_bits():
    """Two graphs and two streams at once, of calls that split their sums: equal bits every time."""
    from megaattention_b200.runtime import linear_int8
    cases = [_case(5, 4096, 512, True), _case(700, 2048, 1280, False, seed=1)]
    want = [linear_int8(*c[:4], bias=c[4]) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(linear_int8(*c[:4], bias=c[4]))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        plain = [linear_int8(*c[:4], bias=c[4]) for c in cases]
        torch.cuda.synchronize()
        for a, b, c in zip(want, outs, plain):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("m", [5, 700])
def test_outputs_that_share_memory_with_an_input(m):
    """Refused, as the inputs are read while outputs are written; columns of one buffer that are the output's alone
    are not."""
    from megaattention_b200.runtime import dequantize_int8, linear_int8
    g = torch.Generator().manual_seed(m)
    room = torch.zeros(m, 4096, dtype=torch.int8, device="cuda")
    x = room[:, :1024]
    x.copy_(_rows(m, 1024, g))
    w, b = _rows(256, 1024, g), torch.randn(256, generator=g).bfloat16().cuda()
    xs, ws = torch.rand(m, generator=g).cuda(), torch.rand(256, generator=g).cuda() / 1000
    wide = room.view(torch.bfloat16)                     # [m, 2048], x in the first 512 of its columns
    before = room.clone()
    for out in (wide[:, :256], wide[:, 511:767], wide[:, 256:512], wide.view(-1)[:m * 256].view(m, 256)):
        with pytest.raises(AssertionError):
            linear_int8(x, xs, w, ws, bias=b, out=out)
    square = torch.zeros(256, 256, dtype=torch.bfloat16, device="cuda")
    scales = square.view(-1).view(torch.float32)[:256]
    call = dict(x=_rows(256, 256, g), x_scale=ws, weight=_rows(256, 256, g), weight_scale=ws, bias=b)
    for kw in (dict(bias=square[2]), dict(weight_scale=scales), dict(x_scale=scales),
               dict(weight=square.view(torch.int8)[:, :256])):
        with pytest.raises(AssertionError):
            linear_int8(**{**call, **kw}, out=square)
    for q, out in ((x, wide[:, :1024]), (room[:, :64], wide[:, 30:94])):
        with pytest.raises(AssertionError):
            dequantize_int8(q, xs, out=out)
    assert torch.equal(room, before)
    _check(linear_int8(x, xs, w, ws, bias=b, out=wide[:, 512:768]), x, xs, w, ws, b)
    assert torch.equal(dequantize_int8(x, xs, out=wide[:, 1024:]), (x.float() * xs[:, None]).bfloat16())
    assert torch.equal(x, before[:, :1024])
