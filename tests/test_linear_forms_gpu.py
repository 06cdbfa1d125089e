"""Every form of the 8-bit projection (csrc/linear_form.h) at a size that takes it: both output types, with and
without a bias, packed rows, and rows of a wider tensor that start at any element, whose surroundings stay as they
are.  That each size takes the form beside it on this GPU's 148 SMs, and that no form is missing here, is checked
without a GPU (tests/test_linear_forms_cpu.py).  Tolerances as in tests/test_linear_int8_gpu.py."""
import pytest
import torch

from test_linear_int8_gpu import _case, _check

pytestmark = pytest.mark.gpu

# (tokens, in, out), (tokens of a tile, stages, parts of K) or (channels of a tile, stages, 0)
FORMS = [
    ((9, 1081, 16893), (16, 6, 1)), ((10, 1002, 7717), (16, 6, 2)), ((9, 1046, 4915), (16, 6, 3)),
    ((16, 1156, 3489), (16, 6, 4)), ((10, 1138, 2599), (16, 6, 6)), ((9, 1430, 12397), (16, 11, 1)),
    ((3, 1073, 6465), (16, 11, 2)), ((9, 4994, 4953), (16, 11, 3)), ((15, 1023, 3411), (16, 11, 4)),
    ((9, 1137, 1001), (16, 11, 6)),
    ((18, 1047, 17627), (32, 5, 1)), ((30, 1147, 9307), (32, 5, 2)), ((17, 1009, 4761), (32, 5, 3)),
    ((20, 1307, 3463), (32, 5, 4)), ((18, 1084, 2665), (32, 5, 6)), ((32, 1119, 12163), (32, 10, 1)),
    ((23, 3557, 9359), (32, 10, 2)), ((20, 259, 133), (32, 10, 3)), ((25, 1230, 3261), (32, 10, 4)),
    ((21, 1047, 1001), (32, 10, 6)),
    ((33, 1036, 23411), (64, 4, 1)), ((36, 1016, 12427), (64, 4, 2)), ((38, 1284, 5987), (64, 4, 3)),
    ((72, 1153, 1781), (64, 4, 4)), ((66, 1087, 1237), (64, 4, 6)), ((36, 16, 11423), (64, 8, 1)),
    ((71, 3333, 4599), (64, 8, 2)), ((41, 1093, 3389), (64, 8, 4)), ((48, 1011, 130), (64, 8, 6)),
    ((540, 1256, 259), (64, 9, 0)), ((1384, 1280, 4097), (128, 7, 0)), ((4000, 512, 5001), (256, 5, 0)),
    ((1111, 4096, 16391), (256, 5, 0)),
]


@pytest.mark.parametrize("size,form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_each_form(size, form, dtype):
    from megaattention_b200.runtime import check_linear_status, linear_int8
    m, k, n = size
    x, xs, w, ws, b = _case(m, k, n, True)
    _check(linear_int8(x, xs, w, ws, out_dtype=dtype), x, xs, w, ws, None)
    _check(linear_int8(x, xs, w, ws, bias=b, out_dtype=dtype), x, xs, w, ws, b)
    whole = -(-n // 8) * 8                               # rows at multiples of 16 bytes whose last 16 are another's too
    for pitch, at in ((n + 1, 1), (n + 9, 7), (whole + 2, 2), (whole + 8, 8), (n + 24, 5)):
        buf = torch.full((m + 1, pitch), -7.0, dtype=dtype, device="cuda")
        out = buf[:m, at:at + n]
        assert linear_int8(x, xs, w, ws, bias=b, out=out) is out
        _check(out, x, xs, w, ws, b)
        out.fill_(-7.0)
        assert bool((buf == -7.0).all())
    check_linear_status()
