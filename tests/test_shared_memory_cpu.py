"""How much dynamic shared memory a kernel may have is raised by whichever thread needs more, and never lowered behind another's back."""
import subprocess

import pytest

HARNESS = r"""
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <thread>
static std::atomic<int> now{0}, calls{0};
static cudaError_t fake_device(int* dev) { *dev = 3; return cudaSuccess; }
template <typename K>
cudaError_t fake_set(K, cudaFuncAttribute, int bytes) {
    if (bytes == 100) std::this_thread::sleep_for(std::chrono::milliseconds(200));     // the smaller one takes its time
    now = bytes;
    ++calls;
    return cudaSuccess;
}
#define cudaFuncSetAttribute fake_set
#define cudaGetDevice fake_device
#include "common.cuh"
__global__ void kernel() {}
int main() {
    bool first = false, second = false;
    std::thread small([&] { first = ti_allow_shared<kernel>(100) == cudaSuccess; });
    std::this_thread::sleep_for(std::chrono::milliseconds(50));
    std::thread large([&] { second = ti_allow_shared<kernel>(200) == cudaSuccess; });
    large.join();
    small.join();
    bool enough = first && second && now >= 200;                                // the launch behind the larger one has what it was given
    const int made = calls;
    enough &= ti_allow_shared<kernel>(150) == cudaSuccess && ti_allow_shared<kernel>(200) == cudaSuccess && calls == made && now >= 200;
    return enough ? 0 : 1;
}
"""


def test_a_smaller_size_does_not_take_a_larger_one_back(tmp_path):
    from tinyinfer_b200.ops import library
    source, program = tmp_path / "harness.cu", tmp_path / "harness"
    source.write_text(HARNESS)
    built = subprocess.run([library.nvcc_path(), *library.ARCH_FLAGS, "-std=c++17", "-I", str(library.CSRC), str(source), "-o", str(program),
                            "-lpthread"], capture_output=True, text=True)
    if built.returncode:
        pytest.fail(built.stderr)
    assert subprocess.run([str(program)], timeout=60).returncode == 0
