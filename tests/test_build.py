"""CPU test of the build's check of register counts: a kernel that shares its
registers out among warpgroups is launched with the number its source is written
for, and a compiler that gives another one fails the build, not the first call."""
import os
import re
import subprocess

import pytest

from quant_2bit_b200 import build

PTXAS = """ptxas info    : 0 bytes gmem
ptxas info    : Compiling entry function '_ZN1a15fp8_rows_kernelI6__halfLi1EEEvi' for 'sm_100a'
ptxas info    : Function properties for _ZN1a15fp8_rows_kernelI6__halfLi1EEEvi
    16 bytes stack frame, 4 bytes spill stores, 12 bytes spill loads
ptxas info    : Used %d registers, used 1 barriers, 16 bytes cumulative stack size
ptxas info    : Compiling entry function '_Z13quantize_rowsPKf' for 'sm_100a'
ptxas info    : Used 58 registers, used 1 barriers
"""


def test_register_counts_are_read_from_ptxas():
    assert build.registers(PTXAS % 168, "fp8_rows_kernel") == [168]
    assert build.registers(PTXAS % 168, "quantize_rows") == [58]
    assert build.registers(PTXAS % 168, "another") == []


def test_another_register_count_fails_the_build(monkeypatch):
    def compile_with(text):
        run = subprocess.CompletedProcess([], 0, stderr=text)
        monkeypatch.setattr(build.subprocess, "run", lambda *a, **k: run)
        build._compile(["nvcc"], "bcjr_fp8.cu", False)

    compile_with(PTXAS % 168)
    for text in (PTXAS % 160, PTXAS.replace("fp8_rows_kernel", "renamed") % 168, ""):
        with pytest.raises(RuntimeError, match="registers"):
            compile_with(text)


def test_every_kernel_that_shares_out_registers_is_checked():
    sources = {n: open(os.path.join(build.CSRC, n)).read() for n in os.listdir(build.CSRC) if n.endswith(".cu")}
    assert {n for n, text in sources.items() if "regs_up<" in text} == set(build.LAUNCH_REGISTERS)
    for name, (kernel, constant) in build.LAUNCH_REGISTERS.items():
        assert kernel in sources[name] and re.search(constant + r" = \d+", sources[name])
