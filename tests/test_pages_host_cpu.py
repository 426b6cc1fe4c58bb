"""The page cache's host code on the CPU (tests/host/pages_host.cpp): qmm_pages.hip compiled against a small stand-in for
the HIP runtime, with allocations and launches that fail on request."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CLANG = shutil.which("clang++", path="/opt/rocm/llvm/bin:" + os.environ.get("PATH", ""))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not CLANG:
        pytest.skip("no clang++ (vector types)")
    out = str(tmp_path_factory.mktemp("host") / "pages_host")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-g", "-Wno-unused", "-I", os.path.join(HERE, "host"),
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "scriptling-llm-lib_amd", "csrc"),
                    os.path.join(HERE, "host", "pages_host.cpp"), "-o", out], check=True)
    return out


@pytest.mark.parametrize("what", ["steps", "refused_begin", "out_of_memory", "failed_copies", "long_sequences", "many_rows"])
def test_host_code(program, what):
    res = subprocess.run([program, what], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
