"""What the compiler may assume of the products of 8-bit rows, in the IR that
the build's own flags give (the GPU is not needed)."""

from __future__ import annotations

import re
import subprocess
from pathlib import Path

import pytest

from titania_amd import build

LDS = "addrspace(3)"


def order_in(body):
    """What a kernel's IR does to LDS from its first ordinary store there on, in
    order: S stores of four f32 or i32, L loads of them, b wave barriers. (The
    loop before fills LDS by direct loads and stores nothing itself.)"""
    steps = ""
    for line in body.splitlines():
        if "llvm.amdgcn.wave.barrier" in line:
            steps += "b"
        elif LDS in line and re.search(r"\bstore <4 x (float|i32)>", line):
            steps += "S"
        elif LDS in line and re.search(r"\bload <4 x (float|i32)>", line):
            steps += "L"
    return steps[steps.find("S"):]


@pytest.mark.skipif(not Path(build.HIPCC).exists(), reason="no HIP compiler")
def test_lanes_that_share_lines_are_ordered(tmp_path):
    """The tiles' results go from lane to lane of a wave through LDS. Every
    change from writing to reading and back stands behind a wave barrier: to
    the compiler another lane's access is free to move otherwise."""
    ir = tmp_path / "q8_matmul.ll"
    flags = [f for f in build.FLAGS if not f.startswith("-Rpass")]
    run = subprocess.run([build.HIPCC, *flags, "--cuda-device-only", "-S", "-emit-llvm", str(build.CSRC / "q8_matmul.hip"),
                          "-o", str(ir)], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    kernels = re.findall(r"^define [^\n]*tile_kernel.*?^}", ir.read_text(), re.S | re.M)
    assert len(kernels) >= 11
    for k in kernels:
        steps, name = order_in(k), re.search(r"TileI\w+?EE", k).group(0)
        assert steps.startswith("S") and steps.endswith("L"), name
        assert "SL" not in steps and "LS" not in steps, (name, steps)
