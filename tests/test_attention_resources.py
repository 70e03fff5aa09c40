"""Resource budgets of the attention kernels, checked at build time from `nvcc
-Xptxas -v` (no GPU).

The tensor-core kernels hand registers from their feeding warps to their
computing ones (setmaxnreg), which waits for ever if the launch does not hold
what is asked for: the launch's registers have to be exactly the 168 (12
warps) or 96 (20 warps) that the split is computed from.  All of L1 is shared
memory there, so a spill goes to L2: none, but for a few words in the backward
with 64 columns (the loop of dk and dv keeps two sums and both operands' addresses)."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


@pytest.mark.skipif(not os.path.exists(NVCC), reason="nvcc absent")
def test_attention_kernels_register_budget(tmp_path):
    src = os.path.join(ROOT, "rushlite_b200", "csrc", "attention_sm100.cu")
    r = subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-Xptxas", "-v",
                        "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "rushlite_b200", "csrc"), "-I",
                        os.path.join(ROOT, "include"), "-c", src, "-o", str(tmp_path / "a.o")], capture_output=True,
                       text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    found, current = {}, None
    for line in r.stderr.splitlines():
        m = re.search(r"Compiling entry function '(\S+)'", line)
        if m:
            k = re.search(r"(forward|backward)_kernelILi(\d+)E", m.group(1))
            current = found.setdefault((k.group(1), int(k.group(2))), {}) if k else None
        if current is None:
            continue
        m = re.search(r"(\d+) bytes spill stores, (\d+) bytes spill loads", line)
        if m:
            current["spill"] = int(m.group(1)) + int(m.group(2))
        m = re.search(r"Used (\d+) registers", line)
        if m:
            current["regs"] = int(m.group(1))
    assert sorted(found) == [(k, d) for k in ("backward", "forward") for d in (64, 128)]
    for (kind, dim), v in found.items():
        assert v["regs"] == (96 if dim == 64 else 168), (kind, dim, v)
        assert v["spill"] <= (128 if (kind, dim) == ("backward", 64) else 0), (kind, dim, v)
