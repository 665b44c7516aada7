"""Private memory of the kernels over 4-bit KV caches, from the metadata of the built libtsr_hip.so: registers that are kept there, and
arrays that the compiler could not keep in registers, cost a decode token a tenth. No GPU calls."""
import glob
import os
import re
import shutil
import subprocess

import pytest

import tsr_hip

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
KERNELS = r"_ZN3tsr\d+(k_attn4\w*?|k_kv4_\w+?|k_kv_pick|k_rope_scaled\w*?)(I\w*?E)?(?:EvN|Ev|PK|EPK)\w*"
# heads of 512, of which no configuration here has any at length; four groups of rows over q4_1
SOME = {"k_attn4ILi512ELi1ELi2ELj2", "k_attn4_blocksILi512ELi2ELj2", "k_attn4_weightsILi128ELi4ELj2", "k_attn4_rowsumsILi128ELi4ELj2"}


def test_private_memory(tmp_path):
    objdump, readelf = os.path.join(LLVM, "llvm-objdump"), os.path.join(LLVM, "llvm-readelf")
    if not (os.path.exists(objdump) and os.path.exists(readelf)):
        pytest.skip("no llvm-objdump / llvm-readelf")
    shutil.copy(tsr_hip.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([objdump, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    sizes = {}
    for co in glob.glob(str(tmp_path / "*gfx950*")):
        notes = subprocess.run([readelf, "--notes", co], check=True, capture_output=True, text=True).stdout
        for name, size in re.findall(r"\.name: +(_ZN3tsr\w+).*?\.private_segment_fixed_size: +(\d+)", notes, re.S):
            if re.match(KERNELS, name):
                sizes[re.sub(r"^_ZN3tsr\d+", "", name)] = int(size)
    assert len(sizes) > 60 and any(k.startswith("k_kv4_scores") for k in sizes) and any(k.startswith("k_attn4_blocks") for k in sizes)
    kept = {k: v for k, v in sizes.items() if v}
    assert all(any(k.startswith(s) for s in SOME) for k in kept), kept
    assert all(v <= (384 if "512" in k else 64) for k, v in kept.items()), kept
