"""What the operators' loads, stores and handovers tell the compiler, seen in what it makes of them. No GPU needed."""
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

HAND = """
#include "operator_common.hip.h"
using namespace cbamd::op;
__global__ void Hand(const float* from, float* to, uint32_t n) {
    __shared__ float words[64];
    words[threadIdx.x] = from[threadIdx.x];
    WaveHandover();
    if (threadIdx.x < n) {
        words[threadIdx.x + 1] = from[64];
    }
    WaveHandover();
    to[threadIdx.x] = words[threadIdx.x];
}
"""


def compiled(tmp_path, text, *flags):
    source, out = tmp_path / "kernel.hip", tmp_path / "kernel.s"
    source.write_text(text)
    subprocess.check_call([HIPCC, "-w", "-x", "hip", "-O3", "-std=c++17"] + build.DEVICE + ["--cuda-device-only", "-S", "-I", CSRC, *flags, str(source), "-o", str(out)],
                          stderr=subprocess.DEVNULL)
    return out.read_text()


@pytest.mark.parametrize("value,bytes_of_it", [("_Float16", 2), ("__bf16", 2), ("uint16_t", 2), ("float", 4), ("double", 8)])
def test_words_of_a_row_are_aligned_as_its_values(tmp_path, value, bytes_of_it):
    """Rows may begin at any value: no access to 16 bytes of 16-bit values may say that they are at a multiple of 4. It is one
    access all the same."""
    accesses = re.findall(r"^.*(?:load|store) .*addrspace\(1\).*align (\d+)", compiled(tmp_path, COPY % (value, value), "-emit-llvm"), re.M)
    assert accesses and all(int(a) <= bytes_of_it for a in accesses)
    assembly = compiled(tmp_path, COPY % (value, value))
    assert assembly.count("global_load_dwordx4") == 1 and assembly.count("global_store_dwordx4") == 1


def test_what_a_wave_hands_over_is_read_again(tmp_path):
    """A lane's own word may be another lane's by then; the stores before the read are not waited for with a barrier or moved."""
    steps = re.findall(r"^\t(ds_write\w*|ds_read\w*|s_barrier|buffer_wbl2|buffer_inv)", compiled(tmp_path, HAND), re.M)
    assert steps == ["ds_write_b32", "ds_write_b32", "ds_read_b32"]
    assert compiled(tmp_path, HAND, "-emit-llvm").count('fence syncscope("wavefront")') == 4
