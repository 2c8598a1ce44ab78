"""What the operators' loads and stores promise the compiler about addresses, seen in what it makes of them. No GPU needed."""
import os
import re
import shutil
import subprocess

import pytest

from catboost_amd import build

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "catboost_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

COPY = """
#include "operator_common.hip.h"
using namespace cbamd::op;
__global__ void Copy(const %s* from, %s* to) {
    TValues<uint32_t, 4>::Load(from + threadIdx.x * 9).Store(to + threadIdx.x * 9);
}
"""


@pytest.mark.parametrize("value,bytes_of_it", [("_Float16", 2), ("__bf16", 2), ("uint16_t", 2), ("float", 4), ("double", 8)])
def test_words_of_a_row_are_aligned_as_its_values(tmp_path, value, bytes_of_it):
    """Rows may begin at any value: no access to 16 bytes of 16-bit values may say that they are at a multiple of 4. It is one
    access all the same."""
    source = tmp_path / "copy.hip"
    source.write_text(COPY % (value, value))
    command = [HIPCC, "-w", "-x", "hip", "-O3", "-std=c++17"] + build.DEVICE + ["--cuda-device-only", "-S", "-I", CSRC, str(source), "-o"]
    subprocess.check_call(command + [str(tmp_path / "copy.ll"), "-emit-llvm"], stderr=subprocess.DEVNULL)
    accesses = re.findall(r"^.*(?:load|store) .*addrspace\(1\).*align (\d+)", (tmp_path / "copy.ll").read_text(), re.M)
    assert accesses and all(int(a) <= bytes_of_it for a in accesses)
    subprocess.check_call(command + [str(tmp_path / "copy.s")], stderr=subprocess.DEVNULL)
    assembly = (tmp_path / "copy.s").read_text()
    assert assembly.count("global_load_dwordx4") == 1 and assembly.count("global_store_dwordx4") == 1
