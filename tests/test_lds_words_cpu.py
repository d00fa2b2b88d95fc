"""Loads of four bytes a lane that write LDS, as they are compiled: five wait states behind a vector write of what they read, one behind m0."""
import re
import shutil
import subprocess

import pytest

from sharpinference_amd.csrc import build as kernel_build
from test_lds_loads_cpu import scalars

SOURCE = r"""
#include "lds_loads.h"
__global__ void words(const char* p, const int* o, int* out, int n) {
  __shared__ __attribute__((aligned(1024))) char smem[4096];
  u32x4 r = buffer_of(p, n);
  load_words_to_lds(r, threadIdx.x * 4, o[threadIdx.x], lds_address(smem));
  r[2] = __builtin_amdgcn_readfirstlane(o[threadIdx.x + 64]);
  load_words_to_lds(r, threadIdx.x * 4, 0, o[threadIdx.x + 128]);
  lds_loads_wait();
  __syncthreads();
  out[threadIdx.x] = *(const int*)(smem + threadIdx.x * 4);
}
"""


def test_a_load_of_words_waits_for_what_it_reads(tmp_path):
    if not (shutil.which("hipcc") or shutil.which("/opt/rocm/bin/hipcc")):
        pytest.skip("hipcc is not installed")
    (tmp_path / "k.hip").write_text(SOURCE)
    subprocess.run([kernel_build._hipcc(), *kernel_build.HIPCC_FLAGS, "-I", kernel_build.CSRC_DIR, "--cuda-device-only", "-S", str(tmp_path / "k.hip"),
                    "-o", str(tmp_path / "k.s")], check=True, stderr=subprocess.DEVNULL)
    ins = [x.split(";")[0].strip() for x in (tmp_path / "k.s").read_text().splitlines() if re.match(r"\s+[svdgb][a-z]*_", x)]
    loads = [i for i, x in enumerate(ins) if x.startswith("buffer_load_dword ") and x.endswith("lds")]
    assert len(loads) == 2
    near = 0
    for i in loads:
        reads, waited = scalars(ins[i]) | {"m0"}, 0
        for x in reversed(ins[:i]):
            if x.startswith("v_read") and scalars(x.split(",")[0]) & reads:
                assert waited >= 5, (x, ins[i], waited)
                near += 1
            if re.match(r"s_mov_b32 m0\b", x):
                assert waited >= 1
            waited += int(x.split()[1]) + 1 if x.startswith("s_nop") else 1
    assert near >= 2
