"""Which form of the 8-bit projection a call takes (csrc/linear_form.h, compiled for the host), and that the GPU
tests of the forms leave none out, however the estimates behind the choice are tuned."""
import ctypes as C
import os
import random
import re
import shutil
import subprocess

import pytest

from test_linear_forms_gpu import FORMS

CSRC = os.path.join(os.path.dirname(__file__), "..", "megaattention_b200", "csrc")
SMS = 148


@pytest.fixture(scope="module")
def form(tmp_path_factory):
    cxx = shutil.which("g++")
    assert cxx, "a C++ compiler is part of the build environment"
    d = tmp_path_factory.mktemp("form")
    (d / "form.cpp").write_text(f'''
#include "{os.path.join(CSRC, "linear_form.h")}"
extern "C" long long form(int tokens, int inner, int width, int sms, int* out) {{
  const ma::LinearForm f = ma::linear_form(tokens, inner, width, sms);
  out[0] = f.width; out[1] = f.stages; out[2] = f.splits;
  return f.tiles;
}}
''')
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o", str(d / "form.so"),
                    str(d / "form.cpp")], check=True, capture_output=True)
    lib = C.CDLL(str(d / "form.so"))
    lib.form.restype = C.c_longlong

    def call(tokens, inner, width, sms=SMS):
        out = (C.c_int * 3)()
        return lib.form(tokens, inner, width, sms, out), tuple(out)

    return call


@pytest.mark.parametrize("size,want", FORMS)
def test_the_sizes_of_the_gpu_tests_take_the_forms_that_they_name(form, size, want):
    assert form(*size)[1] == want


def test_no_form_is_without_a_size(form):
    """Against the forms that the launch can take, read off the source, and those that random sizes take."""
    text = open(os.path.join(CSRC, "linear_quant.cu")).read()
    kernels = {(int(a), int(b)) for a, b in re.findall(r"return launch_(?:narrow|wide)<(\d+), (\d+)>", text)}
    named = {f for _, f in FORMS}
    assert len(kernels) == 9 and {f[:2] for f in named} == kernels
    rng, taken = random.Random(0), {}
    for _ in range(60000):
        size = tuple(round(2 ** rng.uniform(0, top)) for top in (12, 15, 16))
        f = form(*size)[1]
        taken.setdefault(f, []).append(size)
    # (a form that one size in ten thousand takes may stay out)
    assert {f for f, sizes in taken.items() if len(sizes) > 6} <= named, {f: s[:3] for f, s in taken.items() if f not in named}


def test_a_form_fits_its_kernel(form):
    rng = random.Random(1)
    for _ in range(60000):
        size = tuple(round(2 ** rng.uniform(0, top)) for top in (30, 16.99, 30))
        sms = rng.choice([SMS, SMS, 132, 2])
        tiles, (width, stages, splits) = form(*size, sms)
        blocks = (size[1] + 127) // 128
        if splits:
            assert size[0] <= 512 and width in (16, 32, 64) and 1 <= splits <= min(6, blocks)
            assert tiles == -(-size[2] // 128) * -(-size[0] // width) * splits
            assert size[0] <= width or width == 64
        else:
            assert size[0] > 32 and tiles == -(-size[0] // 256) * -(-size[2] // width)
