"""Raising a kernel's shared-memory limit from two threads at once: what is recorded as granted has been granted.  The
CUDA runtime is replaced by two functions of the test; no GPU needed."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "grouped-nf4-gemm_b200" / "csrc"

PROGRAM = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include "api_internal.h"

static std::atomic<int> attribute{0};
static std::atomic<bool> large_set{false}, small_set{false};

static void wait_for(std::atomic<bool>& flag) {          // at most 300 ms: the other thread may be held off
    for (int i = 0; i < 300 && !flag; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
}
extern "C" cudaError_t cudaGetDevice(int* dev) { *dev = 0; return cudaSuccess; }
// the order that used to go wrong: large limit set, small limit set, small one recorded, large one recorded
extern "C" cudaError_t cudaFuncSetAttribute(const void*, enum cudaFuncAttribute, int value) {
    if (value == 200) {
        attribute = value;
        large_set = true;
        wait_for(small_set);
        std::this_thread::sleep_for(std::chrono::milliseconds(50));
    } else {
        wait_for(large_set);
        attribute = value;
        small_set = true;
    }
    return cudaSuccess;
}
static int granted[64];
static void raise(size_t bytes) { gnf4b::ensure_smem(static_cast<const void*>(&attribute), bytes, granted); }
int main() {
    std::thread large(raise, 200), small(raise, 100);
    large.join();
    small.join();
    std::printf("%d %d\n", granted[0], attribute.load());
    return granted[0] == 200 && attribute == 200 ? 0 : 1;
}
"""


def test_two_threads_raise_the_limit(tmp_path):
    cuda = Path(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc").resolve().parent.parent
    gxx = shutil.which("g++")
    if gxx is None or not (cuda / "include" / "cuda_runtime.h").exists():
        pytest.skip("no g++ or no CUDA headers")
    (tmp_path / "main.cpp").write_text(PROGRAM)
    r = subprocess.run([gxx, "-std=c++17", "-pthread", f"-I{CSRC}", f"-I{cuda / 'include'}", "main.cpp", "-o", "main"],
                       cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
