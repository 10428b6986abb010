"""Which of the leaf decoder's kernels have no room for all of their numbers in registers, by the compiler's notes in the built library."""
import os
import re
import shutil
import subprocess

import pytest

from svox_amd.csrc import decoder as D

LLVM = "/opt/rocm/llvm/bin"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """demangled name -> (bytes of memory a lane has for registers it lacks, registers, bytes of LDS)"""
    if not os.path.exists(os.path.join(LLVM, "llvm-readelf")):
        pytest.skip("no LLVM tools")
    at = str(tmp_path_factory.mktemp("library"))
    shutil.copy(D.LIB_PATH, at)
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", os.path.basename(D.LIB_PATH)], cwd=at, check=True, capture_output=True)
    found = {}
    for f in sorted(os.listdir(at)):
        if f.endswith("gfx950"):
            notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", os.path.join(at, f)], check=True, capture_output=True, text=True).stdout
            for kernel in re.split(r"\n\s+- \.agpr_count", notes)[1:]:
                number = lambda key: int(re.search(rf"\.{key}:\s+(\d+)", kernel).group(1))
                found[re.search(r"\.symbol:\s+'?(\S+?)\.kd", kernel).group(1)] = (number("private_segment_fixed_size"), number("vgpr_count"),
                                                                                 number("group_segment_fixed_size"))
    symbols = [s.replace("DF16b", "u6__bf16").replace("DF16_", "Dh") for s in found]     # (the names of types c++filt may not know)
    names = subprocess.run(["c++filt"], input="\n".join(symbols), check=True, capture_output=True, text=True).stdout.split("\n")
    return {re.sub(r"^void |svox_decoder::|\(.*", "", name): found[symbol] for name, symbol in zip(names, found)}


# Weights' gradients of narrow layers in float32, whose three planes of weights and sums are more than 256 registers from 96 features and
# numbers of the result on; the gradients of hidden numbers on large tiles, once a tile, between the products and the results.
LACKING = {r"narrow_weight_kernel<float, (1, 2|2, 1), \d>": 32, r"narrow_weight_kernel<float, 2, 2, \d>": 176,
           r"hidden_kernel<(half|__bf16|_Float16), Shape<256, 128, 64, 2, 4, 2>, true>": 20}


def test_registers_suffice_but_for_what_is_known(kernels):
    assert len(kernels) > 200
    for name, (scratch, registers, lds) in kernels.items():
        most = max([most for pattern, most in LACKING.items() if re.fullmatch(pattern, name)], default=0)
        assert scratch <= most, (name, scratch)
        assert registers <= 256 and lds <= 160 * 1024, name
