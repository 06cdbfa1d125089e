"""The operators' native module: what does without it is there without it, and what needs it says so."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _python(code, **env):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, env={**os.environ, **env}, capture_output=True,
                          text=True, timeout=600)


def test_the_fused_path_is_importable_where_the_module_cannot_be_built(tmp_path):
    got = _python(f'''
from megaattention_b200 import build
build.LIB_CALLS = {str(tmp_path / "_calls.so")!r}
import megaattention_b200.runtime as rt
from megaattention_b200.runtime import FusedFaOprojArWorkspace, FusedPrefillLayer, residual_rmsnorm, rope_qk_
for use in (lambda: rt.rmsnorm_int8(None, None), lambda: rt.linear_int8(None, None, None, None)):
    for _ in range(2):
        try:
            use()
        except ImportError as exc:
            assert "missing and cannot be built" in str(exc), exc
        else:
            raise SystemExit("no ImportError")
print("fine")
''', CXX=str(tmp_path / "no-compiler"))
    assert got.returncode == 0 and got.stdout.strip() == "fine", got.stdout + got.stderr


def test_importing_the_runtime_does_not_load_it():
    got = _python('''
import sys
import megaattention_b200.runtime
assert "megaattention_b200._calls" not in sys.modules
from megaattention_b200 import _native
assert _native.calls is _native.calls and "calls" in vars(_native)
''')
    assert got.returncode == 0, got.stderr
