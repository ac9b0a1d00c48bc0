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
