"""Runs the C++ test program of the decode operators on compressed data
(tests/cpp/test_compressed.cpp), called through include/alpakann_b200/onHost.hpp."""
import subprocess

import pytest


def test_cpp_compressed_builds():
    from tests.cpp import build_compressed
    from tests.helpers import build_library
    build_library()
    assert build_compressed.build()


@pytest.mark.gpu
def test_cpp_compressed_program():
    from tests.cpp import build_compressed
    from tests.helpers import build_library
    build_library()
    r = subprocess.run([build_compressed.build()], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert " 0 failures" in r.stdout
