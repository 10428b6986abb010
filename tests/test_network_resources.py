"""No kernel of the operators of networks over cells lacks registers or LDS, by the compiler's notes in the built library."""
import os
import re
import shutil
import subprocess

import pytest

from svox_amd.csrc import network as N

LLVM = "/opt/rocm/llvm/bin"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """demangled name -> (bytes of memory a lane has for registers it lacks, registers, bytes of LDS)"""
    if not os.path.exists(os.path.join(LLVM, "llvm-readelf")):
        pytest.skip("no LLVM tools")
    at = str(tmp_path_factory.mktemp("library"))
    shutil.copy(N.LIB_PATH, at)
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", os.path.basename(N.LIB_PATH)], cwd=at, check=True, capture_output=True)
    found = {}
    for f in sorted(os.listdir(at)):
        if f.endswith("gfx950"):
            notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", os.path.join(at, f)], check=True, capture_output=True, text=True).stdout
            for kernel in re.split(r"\n\s+- \.agpr_count", notes)[1:]:
                number = lambda key: int(re.search(rf"\.{key}:\s+(\d+)", kernel).group(1))  # noqa: E731
                found[re.search(r"\.symbol:\s+'?(\S+?)\.kd", kernel).group(1)] = (number("private_segment_fixed_size"), number("vgpr_count"),
                                                                                 number("group_segment_fixed_size"))
    symbols = [s.replace("DF16b", "u6__bf16").replace("DF16_", "Dh") for s in found]     # (the names of types c++filt may not know)
    names = subprocess.run(["c++filt"], input="\n".join(symbols), check=True, capture_output=True, text=True).stdout.split("\n")
    return {re.sub(r"^void |svox_network::|\(.*", "", name): found[symbol] for name, symbol in zip(names, found)}


def test_registers_and_lds_suffice(kernels):
    assert len(kernels) > 100
    for name, (scratch, registers, lds) in kernels.items():
        # float32's heads of 128, and gradients of others that go through registers, have a SIMD's registers to themselves, other kernels half of them
        alone = "<float, 128" in name or re.match(r"attend_key_grad_kernel<(float, 64|.*, 128, false)", name)
        assert scratch == 0, (name, scratch)
        assert registers <= (512 if alone or ", 4, " in name else 256) and lds <= 160 * 1024, (name, registers, lds)
