"""The word that kernels report expired waits in: one for a device, however many threads make their first call at a time."""
import os
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <thread>
#include <vector>
#include "status_word.cuh"
static std::atomic<int> made{0}, relaxed{0};
static thread_local cudaStreamCaptureMode mode_now = cudaStreamCaptureModeGlobal;
extern "C" cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode* m) { std::swap(*m, mode_now); return cudaSuccess; }
extern "C" cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) {
    if (made++ == 2) return cudaErrorMemoryAllocation;     // the third one fails
    relaxed += mode_now == cudaStreamCaptureModeRelaxed;
    std::this_thread::sleep_for(std::chrono::milliseconds(50));
    *p = malloc(n);
    *(int*)*p = 77;
    return cudaSuccess;
}
int main() {
    static StatusWords<4> words;
    std::vector<std::thread> all;
    int* got[16];
    for (int i = 0; i < 16; i++) all.emplace_back([&, i] { if (words.get(i & 1, &got[i]) != cudaSuccess || mode_now != cudaStreamCaptureModeGlobal) got[i] = nullptr; });
    for (auto& t : all) t.join();
    std::set<int*> distinct(got, got + 16);
    int* w = nullptr;
    const bool fails = words.get(2, &w) == cudaErrorMemoryAllocation && !w && mode_now == cudaStreamCaptureModeGlobal, then = words.get(2, &w) == cudaSuccess && w;
    printf("%d %d %d %d %d %d\n", (int)distinct.size(), *got[0], *got[1], made.load(), relaxed.load(), fails && then);
}
"""


def test_one_word_a_device(tmp_path):
    (tmp_path / "words.cpp").write_text(PROGRAM)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", f"-I{ROOT / 'c-ml_b200' / 'csrc'}", "-I/usr/local/cuda/include", str(tmp_path / "words.cpp"), "-o", str(tmp_path / "words"),
                    "-lpthread"], check=True, capture_output=True, text=True)
    r = subprocess.run([str(tmp_path / "words")], capture_output=True, text=True, timeout=60)
    assert r.stdout.split() == ["2", "0", "0", "4", "3", "1"], (r.stdout, r.stderr)
