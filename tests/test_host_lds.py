"""How kernels are opted into their LDS sizes (csrc/common.hpp), on the host: the header is compiled against a stand-in for
the HIP runtime that remembers the limit of every kernel and device."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "nerf_amd", "csrc")

RUNTIME = """
#pragma once
#include <cstddef>
#define __host__
#define __device__
#define __global__
enum hipError_t { hipSuccess };
enum { hipFuncAttributeMaxDynamicSharedMemorySize };
hipError_t hipGetDevice(int*);
hipError_t hipFuncSetAttribute(const void*, int, int);
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t) { return ""; }
"""

PROGRAM = """
#include "common.hpp"
#include <atomic>
#include <chrono>
#include <map>
#include <mutex>
#include <thread>

static std::mutex guard;
static std::map<std::pair<const void*, int>, int> limit;
static std::atomic<int> calls{0}, slow_calls{0};
static thread_local int device = 0;
static thread_local bool slow = false;
hipError_t hipGetDevice(int* d) { *d = device; return hipSuccess; }
hipError_t hipFuncSetAttribute(const void* kern, int, int bytes) {
    ++calls;
    if (slow) { ++slow_calls; std::this_thread::sleep_for(std::chrono::milliseconds(300)); }
    std::lock_guard<std::mutex> hold(guard);
    limit[{kern, device}] = bytes;
    return hipSuccess;
}
namespace nerfx {
std::string& last_error_ref() { static std::string s; return s; }
int fail(int code, const char*, ...) { return code; }
}
template <int K> void kernel(int*) {}
static int need(int k, size_t bytes) {
    auto go = [&](auto kern) { NERFX_OPT_IN_LDS(kern, bytes); return 0; };           // one body for kernels of one signature
    return k == 0 ? go(&kernel<0>) : k == 1 ? go(&kernel<1>) : go(&kernel<2>);
}
#define CHECK(...) do { if (!(__VA_ARGS__)) { printf("line %d: %s\\n", __LINE__, #__VA_ARGS__); return 1; } } while (0)
int main() {
    const void* k[3] = {(const void*)&kernel<0>, (const void*)&kernel<1>, (const void*)&kernel<2>};
    // every kernel has a limit of its own, though a larger size was asked for before with another
    CHECK(need(0, 110000) == 0 && limit[{k[0], 0}] == 110000);
    CHECK(need(1, 70000) == 0 && limit[{k[1], 0}] == 70000);
    // never lowered, and not set again
    const int before = calls;
    CHECK(need(0, 70000) == 0 && limit[{k[0], 0}] == 110000 && calls == before);
    CHECK(need(1, 80000) == 0 && limit[{k[1], 0}] == 80000);
    // on each device
    device = 1;
    CHECK(need(0, 66000) == 0 && limit[{k[0], 1}] == 66000 && limit[{k[0], 0}] == 110000);
    // a thread that needs little and is slow, and one that needs much meanwhile
    device = 0;
    int rc = 1;
    std::thread little([&] { slow = true; rc = need(2, 70000); });
    while (slow_calls == 0) std::this_thread::yield();
    CHECK(need(2, 150000) == 0);
    little.join();
    CHECK(rc == 0 && limit[{k[2], 0}] == 150000);
    CHECK(need(2, 140000) == 0 && limit[{k[2], 0}] == 150000);
    return 0;
}
"""


def test_lds_limits_belong_to_kernels_and_never_fall(tmp_path):
    compiler = shutil.which("g++") or shutil.which("clang++")
    if compiler is None:
        pytest.skip("no host compiler")
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text(RUNTIME)
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-O1", "-pthread", f"-I{tmp_path}", f"-I{CSRC}", str(tmp_path / "main.cpp"), "-o",
                    str(tmp_path / "main")], check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout
