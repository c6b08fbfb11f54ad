"""Launchers that want more than 48 KB of shared memory ask for it once a device, against a runtime that counts (no GPU has a part in it)."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "metrale_inference_alpha_b200" / "ops" / "csrc"

PROGRAM = r"""
#include "smem_limit.h"
#include <cstdio>
static int current = 0, calls = 0, fail = 0, last_bytes = 0;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = current; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute a, int bytes) {
  if (a != cudaFuncAttributeMaxDynamicSharedMemorySize) return cudaErrorInvalidValue;
  ++calls;
  last_bytes = bytes;
  return fail ? cudaErrorInvalidValue : cudaSuccess;
}
#define EXPECT(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  std::atomic<uint64_t> a{0}, b{0};
  EXPECT(mb::allow_smem(&a, 70000, a) == cudaSuccess && calls == 1 && last_bytes == 70000);
  EXPECT(mb::allow_smem(&a, 70000, a) == cudaSuccess && calls == 1);          // not again
  EXPECT(mb::allow_smem(&b, 90000, b) == cudaSuccess && calls == 2);          // another kernel
  current = 1;
  EXPECT(mb::allow_smem(&a, 70000, a) == cudaSuccess && calls == 3);          // another device
  EXPECT(mb::allow_smem(&a, 70000, a) == cudaSuccess && calls == 3);
  current = 0;
  EXPECT(mb::allow_smem(&a, 70000, a) == cudaSuccess && calls == 3);
  current = 63, fail = 1;
  EXPECT(mb::allow_smem(&a, 70000, a) != cudaSuccess && calls == 4);          // what failed is not taken as done
  fail = 0;
  EXPECT(mb::allow_smem(&a, 70000, a) == cudaSuccess && calls == 5);
  current = 64;
  EXPECT(mb::allow_smem(&a, 70000, a) == cudaSuccess && mb::allow_smem(&a, 70000, a) == cudaSuccess && calls == 7);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_shared_memory_is_asked_for_once_a_device(tmp_path):
    from metrale_inference_alpha_b200.ops.build import nvcc_path
    include = Path(nvcc_path()).resolve().parent.parent / "include"
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), "-I", str(include), str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_no_launcher_of_these_kernels_keeps_a_flag_for_the_process():
    for name in ("kv_observe.cu", "kv_evict.cu", "kv_mass.cu", "attention_decode_mass.cu", "attention_decode.cuh"):
        assert "cudaFuncSetAttribute" not in (CSRC / name).read_text(), name
