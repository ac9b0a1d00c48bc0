"""What holds for the sources and the host side of the operators on compressed data."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alpakann_b200", "csrc")


def code_of(path):
    """A source file without its comments."""
    with open(path) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", " ", f.read(), flags=re.S)


def test_overlapping_kernels_use_no_read_only_loads():
    """A kernel that is set up while its predecessor still writes may not promise
    that its inputs do not change while it runs."""
    files = [p for p in glob.glob(os.path.join(CSRC, "*.cu")) if '"overlap.cuh"' in code_of(p)]
    assert len(files) >= 4
    for p in files:
        code = code_of(p)
        found = re.findall(r"__ldg\w*|\.nc\b|__restrict(?:__)?\b|__constant__", code)
        assert not found, f"{os.path.basename(p)}: {found}"
        assert "prior_kernels_done()" in code


# ---- the package where the compiled module of the short calls cannot be had ---------
def package_without_module(where):
    """A copy of the package beside the built library alone."""
    import shutil
    pkg = os.path.dirname(CSRC)
    copy = os.path.join(where, "alpakann_b200")
    shutil.copytree(pkg, copy, ignore=shutil.ignore_patterns("_build", "__pycache__", "csrc"))
    os.mkdir(os.path.join(copy, "_build"))
    os.symlink(os.path.join(pkg, "_build", "libann_b200.so"), os.path.join(copy, "_build", "libann_b200.so"))
    return where


REFUSALS = """
import sys
import torch
{before}
import alpakann_b200 as ann
from alpakann_b200 import _short
nn = ann.onHost.nn
assert isinstance(_short.binding, _short.ThroughCtypes) is {fallback}, _short.binding

def refused(error, call, *args, **kw):
    try:
        call(None, None, *args, **kw)
    except error as e:
        return str(e)
    raise AssertionError(f"{{call.__name__}} accepted {{args}}")

i8, i32, f64 = torch.int8, torch.int32, torch.float64
q, c, s = torch.zeros(2, 1, 6, 64), torch.zeros(2, 3, 40, 64, dtype=i8), torch.zeros(2, 3, 3)
assert "kCache" in refused(TypeError, nn.attentionDecodeQ8, q, c.float(), c, s, s, q, 16)
assert "lengths" in refused(TypeError, nn.attentionDecodeQ8, q, c, c, s, s, q, 16, torch.zeros(2, dtype=torch.int64))
assert "CUDA" in refused(ValueError, nn.attentionDecodeQ8, q, c, c, s, s, q, 16)
assert "frequencies" in refused(TypeError, nn.rotary, q, None, torch.zeros(2, 1, dtype=i32), torch.zeros(4), q, None)
assert "CUDA" in refused(ValueError, nn.kvCacheAppendQ8, q[:, :, :3], q[:, :, :3], c, c, s, s, torch.zeros(2, dtype=i32), 16)
assert "kOut" in refused(TypeError, nn.kvCacheReadQ8, c, c, s, s, c, c, 16)
assert "CUDA" in refused(ValueError, nn.linearQ4, torch.zeros(1, 32), torch.zeros(4, 8, dtype=i32), torch.zeros(1, 8),
                         torch.zeros(1, 8), 32)
print("refused")
"""


def run(code, where):
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=where, timeout=300)
    assert r.returncode == 0 and "refused" in r.stdout, r.stdout + r.stderr


def test_the_compiled_module_is_what_runs_here():
    from tests.helpers import ROOT, build_library
    build_library()
    run(REFUSALS.format(before="", fallback=False), ROOT)


def test_package_without_the_compiled_module(tmp_path):
    from tests.helpers import build_library
    build_library()
    run(REFUSALS.format(before="", fallback=True), package_without_module(str(tmp_path)))


def test_package_with_a_torch_without_the_exchange_interface():
    from tests.helpers import ROOT, build_library
    build_library()
    for gone in ("del torch.Tensor.__dlpack_c_exchange_api__", "del torch._C._cuda_getDevice"):
        run(REFUSALS.format(before=gone, fallback=True), ROOT)


def test_package_with_a_module_of_another_build(tmp_path):
    """A file of the module's name that this interpreter cannot load."""
    from tests.helpers import build_library
    build_library()
    from alpakann_b200 import _short
    where = package_without_module(str(tmp_path))
    with open(os.path.join(where, "alpakann_b200", "_build", os.path.basename(_short.PATH)), "wb") as f:
        f.write(b"no shared object")
    run(REFUSALS.format(before="", fallback=True), where)
