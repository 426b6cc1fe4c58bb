"""What a captured batch says of a step that its buffer does not hold (tests/host/outgrown_host.cpp)."""
import os
import subprocess

import pytest

from test_pages_host_cpu import CLANG, HERE, ROOT


@pytest.mark.skipif(not CLANG, reason="no clang++ (vector types)")
def test_host_code(tmp_path):
    out = str(tmp_path / "outgrown_host")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-g", "-Wno-unused", "-I", os.path.join(HERE, "host"),
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "scriptling-llm-lib_amd", "csrc"),
                    os.path.join(HERE, "host", "outgrown_host.cpp"), "-o", out], check=True)
    res = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stderr[-2000:]
