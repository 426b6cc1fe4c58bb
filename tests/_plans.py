"""What a step of a page batch plans, from the host's code alone (host/plan_host.cpp): which blocks of rows the attention's
kernels are given."""
import os
import subprocess
from collections import namedtuple

from test_pages_host_cpu import CLANG, HERE, ROOT

Block = namedtuple("Block", "shape tree causal rows tiles many")
Plan = namedtuple("Plan", "pieces blocks")  # the most pieces of a row (0: none has several)


def compile_program(folder):
    out = os.path.join(str(folder), "plan_host")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-g", "-Wno-unused", "-I", os.path.join(HERE, "host"),
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "scriptling-llm-lib_amd", "csrc"),
                    os.path.join(HERE, "host", "plan_host.cpp"), "-o", out], check=True)
    return out


def plan(program, heads, kv, dk, dtype, page, prefix, owns, rows, parents=None):
    """rows[i] rows for a sequence of owns[i] rows behind a shared prefix; parents: a list for each sequence."""
    line = [heads, kv, dk, int(dtype == "f16"), page, prefix, len(owns), int(parents is not None)]
    for i, (o, n) in enumerate(zip(owns, rows)):
        line += [o, n, *(parents[i] if parents is not None else ())]
    res = subprocess.run([program], input=" ".join(map(str, line)) + "\n", capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    x = [int(v) for v in res.stdout.split()]
    return Plan(x[0], [Block(*x[i:i + 6]) for i in range(1, len(x), 6)])
