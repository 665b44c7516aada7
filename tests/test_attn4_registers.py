"""Registers of the attention over 4-bit KV caches, from the metadata of the built libtsr_hip.so. No GPU calls."""
import glob
import os
import re
import shutil
import subprocess

import pytest

import tsr_hip

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """(head size, row groups, columns a row, type) -> (vector registers, spilled ones)."""
    objdump, readelf = os.path.join(LLVM, "llvm-objdump"), os.path.join(LLVM, "llvm-readelf")
    if not (os.path.exists(objdump) and os.path.exists(readelf)):
        pytest.skip("no llvm-objdump / llvm-readelf")
    tmp = tmp_path_factory.mktemp("co")
    shutil.copy(tsr_hip.LIB_PATH, tmp / "lib.so")
    subprocess.run([objdump, "--offloading", "lib.so"], cwd=tmp, check=True, capture_output=True)
    regs = {}
    for co in glob.glob(str(tmp / "*gfx950*")):
        notes = subprocess.run([readelf, "--notes", co], check=True, capture_output=True, text=True).stdout
        for *form, vgpr, spill in re.findall(r"\.name: +_ZN3tsr7k_attn4ILi(\d+)ELi(\d)ELi(\d)ELj(\d)E\w+.*?\.vgpr_count: +(\d+)"
                                             r".*?\.vgpr_spill_count: +(\d+)", notes, re.S):
            regs[tuple(int(v) for v in form)] = (int(vgpr), int(spill))
    assert len(regs) == 26
    return regs


def test_no_spills(kernels):
    """Nothing is kept in memory, but by one kernel for heads of 512."""
    assert {k for k, (_, spill) in kernels.items() if spill} <= {(512, 1, 2, 2)}
    assert kernels[512, 1, 2, 2][1] <= 80


def test_waves(kernels):
    """Four waves a SIMD (128 registers) for heads of 64 with one group of rows, three (168) for a token's heads of 128, two for
    the rest up to heads of 256."""
    for (D, NT, C, typ), (vgpr, _) in kernels.items():
        most = 128 if D * NT == 64 else 168 if (D, C) == (128, 4) else 256 if D <= 256 else 512
        assert vgpr <= most, (D, NT, C, typ, vgpr)
