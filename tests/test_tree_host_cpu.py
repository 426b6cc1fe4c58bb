"""Steps of drafted trees, the host's part, on the CPU (tests/host/tree_host.cpp): qmm_pages.hip compiled against a small
stand-in for the HIP runtime."""
import os
import subprocess

import pytest

from test_pages_host_cpu import CLANG, HERE, ROOT


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not CLANG:
        pytest.skip("no clang++ (vector types)")
    out = str(tmp_path_factory.mktemp("host") / "tree_host")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-g", "-Wno-unused", "-I", os.path.join(HERE, "host"),
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "scriptling-llm-lib_amd", "csrc"),
                    os.path.join(HERE, "host", "tree_host.cpp"), "-o", out], check=True)
    return out


@pytest.mark.parametrize("what", ["steps", "refused"])
def test_host_code(program, what):
    res = subprocess.run([program, what], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
