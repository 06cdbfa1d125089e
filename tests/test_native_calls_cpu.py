"""The operators' native module: what does without it is there without it, and what needs it says so."""
import os
import shutil
import subprocess
import sys
import sysconfig

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _python(code, cwd=ROOT, **env):
    return subprocess.run([sys.executable, "-c", code], cwd=cwd, env={**os.environ, **env}, capture_output=True,
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
from megaattention_b200 import _native
assert "calls" not in vars(_native)
assert _native.calls is _native.calls and "calls" in vars(_native)
''')
    assert got.returncode == 0, got.stderr


@pytest.mark.parametrize("entry", ["import", "build"])
def test_a_module_of_another_torch_is_not_used(tmp_path, entry):
    """What another torch's build left beside the package, newer than every source, is neither loaded nor taken
    for this one's: the module is built again (by a compiler that hands out the one that is there)."""
    from megaattention_b200 import build
    from megaattention_b200._native import calls
    here = tmp_path / "megaattention_b200"
    shutil.copytree(os.path.join(ROOT, "megaattention_b200"), here, ignore=shutil.ignore_patterns("_calls*", "__pycache__"))
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    shutil.copy(os.path.join(ROOT, "__graft_entry__.py"), tmp_path)
    for lib in here.glob("*.so"):
        os.utime(lib)
    for name in ("_calls", "_calls_torch0.0.0"):
        (here / (name + sysconfig.get_config_var("EXT_SUFFIX"))).write_bytes(b"of another torch")
    cxx = tmp_path / "cxx"
    cxx.write_text(f"""#!/bin/sh
while [ $# -gt 1 ]; do if [ "$1" = -o ]; then cp {build.LIB_CALLS} "$2"; fi; shift; done
echo built >> {tmp_path}/log
""")
    cxx.chmod(0o755)
    got = _python("import __graft_entry__ as g; g.build()\n" * (entry == "build") + f"""
import torch
from megaattention_b200 import _native, build
assert build.HERE == {str(here)!r}, build.HERE
assert _native.calls.torch_version == torch.__version__ == build.torch_version()
""", cwd=tmp_path, CXX=str(cxx))
    assert got.returncode == 0, got.stderr
    assert (tmp_path / "log").read_text() == "built\n"
    assert calls.torch_version in os.path.basename(build.LIB_CALLS)


@pytest.mark.parametrize("home", [False, True])
def test_cuda_headers_are_those_of_the_compiler_on_the_path(tmp_path, home):
    """As for the kernels: a toolkit anywhere, if its nvcc is on the path, or CUDA_HOME."""
    (tmp_path / "toolkit" / "bin").mkdir(parents=True)
    (tmp_path / "toolkit" / "bin" / "nvcc").write_text("#!/bin/sh\n")
    cxx = tmp_path / "cxx"
    cxx.write_text(f"#!/bin/sh\necho \"$@\" > {tmp_path}/log\nexit 1\n")
    for f in (cxx, tmp_path / "toolkit" / "bin" / "nvcc"):
        f.chmod(0o755)
    env = dict(CXX=str(cxx), PATH=f"{tmp_path}/toolkit/bin:{os.environ['PATH']}", CUDA_HOME=str(tmp_path / "home") if home else "")
    got = _python(f"""
from megaattention_b200 import build
build.LIB_CALLS = {str(tmp_path / "_calls.so")!r}
try:
    build.build_calls()
except RuntimeError:
    print("refused")
""", NVCC="nvcc", **env)
    assert got.stdout.strip() == "refused", got.stderr
    assert f"-I{tmp_path}/{'home' if home else 'toolkit'}/include " in (tmp_path / "log").read_text()


@pytest.mark.parametrize("version", ["__version__ = '7.1.2+cu999'", '__version__: str = "7.1.2+cu999"', "import os", None])
def test_the_version_of_torch_is_found_wherever_it_stands(tmp_path, version):
    """Importing the package does without importing torch only if it can."""
    (tmp_path / "torch").mkdir()
    (tmp_path / "torch" / "__init__.py").write_text("__version__ = '7.1.2+cu999'\n")
    if version is not None:
        (tmp_path / "torch" / "version.py").write_text(f"from typing import Optional\n{version}\ncuda = '12.8'\n")
    got = _python("""
import sys
from megaattention_b200 import build
print(build.torch_version(), "_calls_torch7.1.2+cu999." in build.LIB_CALLS, "torch" in sys.modules)
""", PYTHONPATH=str(tmp_path))
    assert got.stdout.split() == ["7.1.2+cu999", "True", str(version is None or "version" not in version)], got.stderr
