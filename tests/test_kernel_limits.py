"""Shared memory above 48 KB is asked for on every device that a process uses, and once on each."""
import os
import re
import shutil
import subprocess

import pytest

from photon_infer_b200.csrc.build import CSRC_DIR, find_nvcc

SMALL_CACHES = ("cache_evict", "key_weights", "key_weights_rows", "key_weights_mma", "key_weights_tc", "kv4", "kv4_attention", "kv4_attention_rows", "kv4_attention_mma")

HARNESS = r"""
#include "limits.cuh"
#include <stdio.h>
static int now, asked[128][2], fail;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = now; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute what, int value) {
  if (fail) return cudaErrorInvalidValue;
  ++asked[now][what == cudaFuncAttributePreferredSharedMemoryCarveout];
  return value > 0 ? cudaSuccess : cudaErrorInvalidValue;
}
int main() {
  static bool ready[64], other[64];
  int bad = 0;
  fail = 1; now = 3; bad += smem_limit(0, 1000, true, ready) == 0; fail = 0;      // a call that failed is made again
  for (int round = 0; round < 3; ++round)
    for (now = 0; now < 70; ++now) bad += smem_limit(0, 1000, true, ready) != 0;
  now = 5; bad += smem_limit(0, 1000, false, other) != 0;
  for (int d = 0; d < 64; ++d) bad += asked[d][0] != (d == 5 ? 2 : 1) || asked[d][1] != 1;
  bad += asked[69][0] != 3;                                                          // beyond the table: every time
  printf("%d\n", bad);
  return bad;
}
"""


def test_once_a_device(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "harness.cpp").write_text(HARNESS)
    cuda = os.path.dirname(os.path.dirname(find_nvcc()))
    subprocess.run([cxx, "-std=c++17", "-I", CSRC_DIR, "-I", os.path.join(cuda, "include"), str(tmp_path / "harness.cpp"), "-o", str(tmp_path / "harness")], check=True)
    assert subprocess.run([str(tmp_path / "harness")], capture_output=True, text=True).stdout == "0\n"


@pytest.mark.parametrize("module", SMALL_CACHES)
def test_nothing_is_set_once_a_process(module):
    with open(os.path.join(CSRC_DIR, module + ".cu")) as f:
        source = f.read()
    assert "cudaFuncSetAttribute" not in source and not re.search(r"static\s+bool\s+\w+\s*=", source)
