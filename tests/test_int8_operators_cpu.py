"""The operators between two layers without a GPU: what their C entry points refuse before any
device call, their structs' layout, the place of a step's rows in a paged cache, weights in 8 bits."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest
import torch

from megaattention_b200 import _cabi
from megaattention_b200.runtime import quantize_weight_int8
from oracle.int8_oracle import rmsnorm_int8_oracle, rope_append_oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MB = 1 << 20
BAD, FULL, OK = _cabi.MA_ERR_INVALID, _cabi.MA_ERR_CAPACITY, _cabi.MA_OK


def _calls(fn, struct, ok):
    assert fn(None, None) == BAD
    return lambda **kw: fn(C.byref(struct(**{**ok, **kw})), None)


def test_norm_refuses_before_any_device_call():
    ok = dict(x=MB, residual_in=2 * MB, weight=3 * MB, residual_out=4 * MB, q_out=5 * MB, scale_out=6 * MB,
              x_pitch=1024, residual_in_pitch=1024, residual_out_pitch=1024, q_pitch=1024, rows=0, hidden=1024,
              eps=1e-6)
    call = _calls(_cabi.lib.ma_rmsnorm_quant, _cabi.RmsNormQuantArgs, ok)
    assert call() == OK                                              # nothing to do
    assert call(residual_in=0, residual_out=0) == OK
    for kw in (dict(x=0), dict(weight=0), dict(q_out=0), dict(scale_out=0), dict(residual_in=0),
               dict(residual_out=0), dict(x=MB + 8), dict(weight=MB + 2), dict(q_out=MB + 8), dict(scale_out=MB + 2),
               dict(residual_in=MB + 8), dict(residual_out=MB + 4), dict(rows=-1), dict(hidden=0), dict(hidden=1020),
               dict(eps=-1e-6), dict(eps=float("nan")), dict(x_pitch=1016), dict(x_pitch=1028), dict(q_pitch=1016),
               dict(q_pitch=1032), dict(residual_in_pitch=512), dict(residual_out_pitch=1025), dict(cu_q=MB),
               dict(fa_b=MB, fa_mb=MB)):
        assert call(**kw) == BAD, kw
    wide = dict(hidden=16392, x_pitch=16392, residual_in_pitch=16392, residual_out_pitch=16392, q_pitch=16400)
    assert call(**wide) == FULL
    assert call(rows=(1 << 30) + 1) == FULL
    assert call(rows=(1 << 23) + 1, cu_q=MB, fa_b=MB, fa_mb=MB) == FULL


def test_linear_refuses_before_any_device_call():
    ok = dict(x=MB, weight=2 * MB, x_scale=3 * MB, weight_scale=4 * MB, bias=0, out=5 * MB, x_pitch=1008,
              weight_pitch=1008, out_pitch=1001, tokens=0, inner=1000, width=1001, out_f32=0)
    call = _calls(_cabi.lib.ma_linear_quant, _cabi.LinearQuantArgs, ok)
    assert call() == OK and call(tokens=3, width=0) == OK            # nothing to do
    for kw in (dict(x=0), dict(weight=0), dict(x_scale=0), dict(weight_scale=0), dict(out=0), dict(x=MB + 8),
               dict(weight=MB + 8), dict(x_pitch=1000), dict(x_pitch=992), dict(weight_pitch=1004), dict(out_pitch=1000),
               dict(tokens=-1), dict(width=-1), dict(inner=0), dict(x_scale=MB + 2), dict(weight_scale=MB + 1),
               dict(bias=MB + 1), dict(out=MB + 1), dict(out=MB + 2, out_f32=1)):
        assert call(**kw) == BAD, kw
    assert call(inner=131072, x_pitch=131072, weight_pitch=131072) == FULL       # sums could pass 32 bits
    assert _cabi.lib.ma_linear_status(None, None) == BAD


def test_append_refuses_before_any_device_call():
    ok = dict(q=MB, k=2 * MB, v=3 * MB, out=4 * MB, k_cache=5 * MB, v_cache=6 * MB, cu_q=7 * MB, cache_seqlens=8 * MB,
              page_table=9 * MB, inv_freq=10 * MB, dropped=0, q_tok=1024, q_head=128, k_tok=128, k_head=128, v_tok=128,
              v_head=128, out_tok=1024, out_head=128, table_pitch=7, rows=0, num_batch=3, H_local=8, H_kv=1,
              num_pages=9, table_width=7)
    call = _calls(_cabi.lib.ma_rope_append, _cabi.RopeAppendArgs, ok)
    assert call() == OK
    for name in ("q", "k", "v", "out", "k_cache", "v_cache"):
        assert call(**{name: 0}) == BAD and call(**{name: MB + 8}) == BAD
    for name in ("cu_q", "cache_seqlens", "page_table", "inv_freq"):
        assert call(**{name: 0}) == BAD and call(**{name: MB + 2}) == BAD
    for kw in (dict(dropped=MB + 2), dict(q_tok=1020), dict(k_head=-128), dict(out_head=4), dict(table_pitch=6),
               dict(rows=-1), dict(num_batch=0), dict(H_local=0), dict(H_kv=0), dict(num_pages=0),
               dict(table_width=0)):
        assert call(**kw) == BAD, kw
    assert call(rows=(1 << 30) + 1) == FULL


def test_dequantizing_refuses_before_any_device_call():
    ok = dict(q=MB, scale=2 * MB, out=3 * MB, q_pitch=1008, out_pitch=1000, rows=0, cols=1000, out_f32=0)
    call = _calls(_cabi.lib.ma_dequant, _cabi.DequantArgs, ok)
    assert call() == OK and call(rows=4, cols=0) == OK
    for kw in (dict(q=0), dict(scale=0), dict(out=0), dict(q=MB + 8), dict(scale=MB + 2), dict(out=MB + 1),
               dict(out=MB + 2, out_f32=1), dict(q_pitch=992), dict(q_pitch=1004), dict(out_pitch=999), dict(rows=-1),
               dict(cols=-1)):
        assert call(**kw) == BAD, kw


def test_structs_agree_with_the_compiled_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    assert cc, "a C compiler is part of the build environment"
    pairs = {"ma_rmsnorm_quant_args": _cabi.RmsNormQuantArgs, "ma_linear_quant_args": _cabi.LinearQuantArgs,
             "ma_rope_append_args": _cabi.RopeAppendArgs, "ma_dequant_args": _cabi.DequantArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>',
             '#include "%s"' % os.path.join(ROOT, "include", "megaattn_b200.h"), 'int main(void) {']
    want = []
    for cname, ct in pairs.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % cname)
        want.append(C.sizeof(ct))
        for f, _ in ct._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (cname, f))
            want.append(getattr(ct, f).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run([cc, "-std=c99", "-o", str(exe), str(src)], check=True, capture_output=True)
    got = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


@pytest.fixture(scope="module")
def place(tmp_path_factory):
    """The kernel's own search and bounds checks (csrc/append_place.h), compiled for the host: 32 lanes'
    probes one after the other, every index that is read checked against its array."""
    cxx = shutil.which("g++")
    assert cxx, "a C++ compiler is part of the build environment"
    d = tmp_path_factory.mktemp("place")
    (d / "place.cpp").write_text('''
#include "%s"
extern "C" int place(const int* cu_q, int num_batch, int t, const int* lens, const int* table, int pitch, int width,
                     int num_pages, int* pos, int* page) {
  int lo = 0, n = num_batch, rounds = 0;
  while (n > 1) {
    int hits = 0;
    for (int lane = 0; lane < 32; ++lane) {
      const int at = lane * ma::search_step(n);
      const int i = lo + (at < n ? at : 0);
      if (i < 0 || i > num_batch) return -100;
      hits += at < n && cu_q[i] <= t;
    }
    ma::search_take(hits, &lo, &n);
    if (n < 1 || lo < 0 || lo + n > num_batch || ++rounds > 8) return -101;
  }
  *pos = ma::position_of(t, cu_q[lo], cu_q[lo + 1], lens[lo]);
  *page = ma::page_of(*pos, table + static_cast<long long>(lo) * pitch, width, num_pages);
  return lo;
}
''' % os.path.join(ROOT, "megaattention_b200", "csrc", "append_place.h"))
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-o", str(d / "place.so"), str(d / "place.cpp")],
                   check=True, capture_output=True)
    lib = C.CDLL(str(d / "place.so"))

    def call(cu_q, t, lens, table, width, num_pages):
        nb = len(lens)
        a = (C.c_int * len(cu_q))(*cu_q)
        b = (C.c_int * nb)(*lens)
        c = (C.c_int * (nb * width))(*[x for row in table for x in row])
        pos, page = C.c_int(), C.c_int()
        at = lib.place(a, nb, t, b, c, width, width, num_pages, C.byref(pos), C.byref(page))
        return at, pos.value, page.value

    return call


@pytest.mark.parametrize("batch", [1, 2, 31, 32, 33, 63, 64, 65, 700, 1024, 1025, 3000])
def test_every_row_finds_its_sequence(place, batch):
    rng = random.Random(batch)
    for empty in (0.0, 0.5, 0.95):
        lens_q = [0 if rng.random() < empty else rng.randint(1, 5) for _ in range(batch)]
        if not sum(lens_q):
            lens_q[-1 if batch % 2 else 0] = 3
        lens_k = [n + rng.randint(0, 300) for n in lens_q]
        cu = [0]
        for n in lens_q:
            cu.append(cu[-1] + n)
        table = [[rng.randint(0, 49) for _ in range(3)] for _ in lens_q]
        owner = [b for b, n in enumerate(lens_q) for _ in range(n)]
        for t in sorted({0, cu[-1] - 1} | {rng.randrange(cu[-1]) for _ in range(40)}):
            b = owner[t]
            pos = lens_k[b] - (cu[b + 1] - t)
            assert place(cu, t, lens_k, table, 3, 50) == (b, pos, table[b][pos // 128])


def test_rows_without_a_place_have_none(place):
    cu, table = [0, 4, 8], [[5, 6], [7, 99]]
    assert place(cu, 0, [4, 300], table, 2, 99) == (0, 0, 5)
    assert place(cu, 0, [3, 300], table, 2, 99) == (0, -1, -1)          # before the first key
    assert place(cu, 1, [3, 300], table, 2, 99) == (0, 0, 5)
    assert place(cu, 3, [0, 300], table, 2, 99)[1:] == (-1, -1)         # a sequence without keys
    assert place(cu, 3, [-2 ** 31, 300], table, 2, 99)[1:] == (-1, -1)
    assert place(cu, 7, [4, 200], table, 2, 99) == (1, 199, -1)         # page 99 of 99
    assert place(cu, 7, [4, 200], [[5, 6], [7, -1]], 2, 99) == (1, 199, -1)
    assert place(cu, 7, [4, 200], table, 2, 100) == (1, 199, 99)
    assert place(cu, 7, [4, 257], table, 2, 100) == (1, 256, -1)        # past the table
    assert place(cu, 7, [4, 2 ** 31 - 1], table, 2, 100)[2] == -1
    assert place([2, 4, 8], 0, [4, 4], table, 2, 100)[1] == -1          # before the first sequence
    for bad in ([0, -7, 8], [0, 2 ** 31 - 1, 8], [-2 ** 31, 4, 8], [8, 4, 0]):   # not ascending: no wild index
        for t in (0, 3, 7):
            b, pos, page = place(bad, t, [4, 4], table, 2, 100)
            assert b in (0, 1) and page in (-1, 5, 6, 7, 99)


def test_calls_refuse_what_is_not_on_a_gpu():
    """The native checks (csrc/calls.cpp) on host tensors, and arguments that are no tensors at all."""
    from megaattention_b200._native import calls
    from megaattention_b200.runtime import dequantize_int8, linear_int8, rmsnorm_int8, rope_append
    x, w = torch.ones(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    q, s = torch.ones(4, 64, dtype=torch.int8), torch.ones(4)
    i = torch.ones(2, dtype=torch.int32)
    h = torch.ones(1, 2, 128, dtype=torch.bfloat16)
    for bad in (lambda: rmsnorm_int8(x, w), lambda: rmsnorm_int8([1.0], w), lambda: rmsnorm_int8(x, None),
                lambda: linear_int8(q, s, q, s), lambda: linear_int8(None, s, q, s), lambda: dequantize_int8(q, s),
                lambda: rope_append(h, h, h, h, h, i[None], i, i, inv_freq=s), lambda: rope_append(h, 3, h, h, h, i, i, i)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        calls.linear_int8(q, s)
    with pytest.raises(TypeError):
        linear_int8(q, s, q)
    assert calls.torch_version == torch.__version__


def test_weights_in_eight_bits():
    g = torch.Generator().manual_seed(5)
    for n, k, dtype in ((7, 100, torch.float32), (16, 64, torch.bfloat16), (3, 1, torch.float32)):
        w = torch.randn(n, k, generator=g).to(dtype)
        w[1] = 0
        q, s = quantize_weight_int8(w)
        assert q.shape == (n, k) and q.dtype == torch.int8 and q.stride(0) % 16 == 0
        assert s.shape == (n,) and s.dtype == torch.float32
        # half a step, and fp32's roundings of the quotient (|q| <= 127, three of them)
        step = s.double()[:, None]
        assert bool(((q.double() * step - w.double()).abs() <= step * (0.5 + 127 * 3 * 2.0 ** -24)).all())
        assert float(s[1]) == 0 and int(q[1].abs().max()) == 0
        assert bool((q[w.abs().amax(1) > 0].abs().amax(1) == 127).all())


def test_oracles_agree_with_other_statements_of_the_same():
    g = torch.Generator().manual_seed(6)
    x, w = torch.randn(5, 64, generator=g).to(torch.bfloat16), torch.randn(64, generator=g).to(torch.bfloat16)
    t, scale, h = rmsnorm_int8_oracle(x, w, 1e-5)
    ref = torch.nn.functional.rms_norm(x.double(), (64,), w.double(), 1e-5)
    assert torch.allclose(t * scale[:, None], ref, rtol=1e-12, atol=0) and h is x
    from oracle.producer_oracle import inv_freq_fp32, rope_oracle
    q, k = torch.randn(6, 2, 128, generator=g).to(torch.bfloat16), torch.randn(6, 1, 128, generator=g).to(torch.bfloat16)
    cache = torch.zeros(3, 128, 1, 128, dtype=torch.bfloat16)
    out, kc, vc, _, _, dropped = rope_append_oracle(q, k, k, cache, cache, [[2], [0]], [2, 4], [0, 2, 6], inv_freq_fp32())
    qo, ko = rope_oracle(q, k, [2, 4])
    assert dropped == 0 and torch.allclose(out, qo.double(), rtol=2.0 ** -7, atol=1e-5)
    assert torch.allclose(torch.cat([kc[2, :2], kc[0, :4]]), ko.double(), rtol=2.0 ** -7, atol=1e-5)
    assert torch.equal(torch.cat([vc[2, :2], vc[0, :4]]), k) and not bool(vc[1].any())


def test_every_row_of_a_batch_that_fits_a_warp_finds_its_sequence(tmp_path):
    """The kernel's other way to a row's sequence (csrc/append_place.h): 32 lanes' loads one after the other, every
    index checked, and the two shuffles from the lanes that they name."""
    cxx = shutil.which("g++")
    assert cxx, "a C++ compiler is part of the build environment"
    (tmp_path / "small.cpp").write_text('''
#include "%s"
extern "C" int most() { return ma::kSmallBatch; }
extern "C" int small(const int* cu_q, int num_batch, int t, const int* lens, int* got) {
  int start[32], keys[32], hits = 0;
  for (int lane = 0; lane < 32; ++lane) {
    const int i = ma::small_start(lane, num_batch), j = ma::small_keys(lane, num_batch);
    if (i < 0 || i > num_batch || j < 0 || j >= num_batch) return -100;
    start[lane] = cu_q[i];
    keys[lane] = lens[j];
    hits += lane < num_batch && start[lane] <= t;
  }
  const int b = ma::small_take(hits);
  if (b < 0 || b + 1 > 31) return -101;
  got[0] = start[b]; got[1] = start[b + 1]; got[2] = keys[b];
  return b;
}
''' % os.path.join(ROOT, "megaattention_b200", "csrc", "append_place.h"))
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-o", str(tmp_path / "small.so"),
                    str(tmp_path / "small.cpp")], check=True, capture_output=True)
    lib = C.CDLL(str(tmp_path / "small.so"))
    assert lib.most() == 31                  # (lane b + 1 is there for the last of them)
    rng = random.Random(7)
    for _ in range(300):
        nb = rng.choice([1, 2, 5, 30, 31])
        empty = rng.choice([0.0, 0.5, 0.95])
        lens_q = [0 if rng.random() < empty else rng.randint(1, 5) for _ in range(nb)]
        lens = (C.c_int * nb)(*[rng.randint(0, 900) for _ in range(nb)])
        cu = [0]
        for n in lens_q:
            cu.append(cu[-1] + n)
        owner = [b for b, n in enumerate(lens_q) for _ in range(n)]
        for t in range(cu[-1]):
            got = (C.c_int * 3)()
            b = lib.small((C.c_int * (nb + 1))(*cu), nb, t, lens, got)
            assert b == owner[t] and list(got) == [cu[b], cu[b + 1], lens[b]]
    for bad in ([0, -7, 8], [0, 2 ** 31 - 1, 8], [-2 ** 31, 4, 8], [8, 4, 0], [2, 4, 8]):     # no wild index
        for t in (0, 3, 7):
            assert lib.small((C.c_int * 3)(*bad), 2, t, (C.c_int * 2)(4, 4), (C.c_int * 3)()) in (0, 1)
