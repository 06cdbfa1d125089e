"""A bounded wait of the 8-bit projection that runs out: the call ends by itself with every copy landed, the
status says where it gave up, once, and the next call is right.

The audit build's issuers wait, at a given block of K, for a barrier that nobody arrives at (and for 0.2 s
instead of 2); everything else is as in the product.  Nothing traps."""
import ctypes as C
import threading

import pytest
import torch

from megaattention_b200 import _cabi
from oracle.int8_oracle import linear_int8_oracle

pytestmark = pytest.mark.gpu


@pytest.fixture()
def audit():
    lib = _cabi.audit_lib()
    lib.ma_audit_linear_stall.argtypes = [C.c_int]
    lib.ma_audit_linear_stall.restype = None
    lib.ma_audit_linear_stall(-1)
    assert _counts(lib)[2] >= 0
    yield lib
    lib.ma_audit_linear_stall(-1)
    torch.cuda.synchronize()
    _status(lib)


def _counts(lib):
    n = (C.c_uint32 * 3)()
    assert lib.ma_audit_linear_counts(n) == _cabi.MA_OK
    return list(n)


def _status(lib):
    st = _cabi.Status()
    rc = lib.ma_linear_status(torch.cuda.current_stream().cuda_stream, C.byref(st))
    return rc, st


def _case(m, k, n):
    g = torch.Generator().manual_seed(m + k + n)
    x = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8).cuda()
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda()
    return x, torch.rand(m, generator=g).cuda() + 0.01, w, torch.rand(n, generator=g).cuda() / 1000


def _run(lib, x, xs, w, ws, out):
    (m, k), n = x.shape, w.shape[0]
    a = _cabi.LinearQuantArgs(x=x.data_ptr(), weight=w.data_ptr(), x_scale=xs.data_ptr(), weight_scale=ws.data_ptr(),
                              bias=0, out=out.data_ptr(), x_pitch=k, weight_pitch=k, out_pitch=n, tokens=m, inner=k,
                              width=n, out_f32=int(out.dtype == torch.float32))
    assert lib.ma_linear_quant(C.byref(a), torch.cuda.current_stream().cuda_stream) == _cabi.MA_OK
    torch.cuda.synchronize()


# few tokens with one part of K and several, shorter than the ring and longer; many tokens in three widths
CASES = [(5, 512, 300, 3), (5, 4096, 512, 0), (5, 4096, 512, 31), (20, 8192, 1000, 17), (48, 16384, 256, 127),
         (60, 1024, 40000, 7), (700, 2048, 1280, 0), (700, 2048, 1280, 15), (4100, 256, 1000, 1), (2049, 1152, 4096, 8)]


@pytest.mark.parametrize("m,k,n,block", CASES)
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(audit, m, k, n, block):
    x, xs, w, ws = _case(m, k, n)
    out = torch.full((m, n), 3.0, device="cuda")
    _counts(audit)
    audit.ma_audit_linear_stall(block)
    _run(audit, x, xs, w, ws, out)
    audit.ma_audit_linear_stall(-1)
    waited, landed, gave_up = _counts(audit)
    assert gave_up > 0 and waited > 0 and landed == waited, (waited, landed, gave_up)
    rc, st = _status(audit)
    assert rc == _cabi.MA_ERR_DEVICE_TIMEOUT and st.code != 0 and st.site in (0x10, 0x12, 0x13, 0x20, 0x22, 0x23, 0x24)
    assert _status(audit)[0] == _cabi.MA_OK                    # said once
    _run(audit, x, xs, w, ws, out)
    ref, size = linear_int8_oracle(x, xs, w, ws)
    # (as in tests/test_linear_int8_gpu.py: conversion, two products, and the result's rounding)
    assert bool(((out.double() - ref).abs() <= 5 * 2.0 ** -24 * size).all())
    assert _status(audit)[0] == _cabi.MA_OK and _counts(audit) == [0, 0, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,n,block", CASES)
def test_what_was_not_computed_is_nan(audit, m, k, n, block, dtype):
    """Every tile lacks a block of its sum, or its pair of CTAs gave up before it; nothing behind the output changes."""
    x, xs, w, ws = _case(m, k, n)
    buf = torch.full((m + 1, n), 3.0, device="cuda", dtype=dtype)
    audit.ma_audit_linear_stall(block)
    _run(audit, x, xs, w, ws, buf[:m])
    assert bool(buf[:m].isnan().all()) and bool((buf[m] == 3).all())


def test_one_of_many_who_ask_at_once_gets_the_report(audit):
    """A single CTA gives up: a single report, to whoever is first."""
    x, xs, w, ws = _case(3, 128, 100)
    out = torch.empty(3, 100, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(8)]
    for _ in range(5):
        audit.ma_audit_linear_stall(0)
        _run(audit, x, xs, w, ws, out)
        audit.ma_audit_linear_stall(-1)
        start, got = threading.Barrier(len(streams)), []

        def ask(stream):
            st = _cabi.Status()
            start.wait()
            got.append(audit.ma_linear_status(stream.cuda_stream, C.byref(st)))

        threads = [threading.Thread(target=ask, args=(s,)) for s in streams]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert sorted(got) == [_cabi.MA_ERR_DEVICE_TIMEOUT] + [_cabi.MA_OK] * 7
