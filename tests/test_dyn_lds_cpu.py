"""csrc/dyn_lds.h on the host, against a runtime of several devices that counts its calls: a
kernel's LDS limit holds on the device it was set on, and a smaller one never follows a larger."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

PROGRAM = r"""
#include "dyn_lds.h"
#include <cstdio>
#include <thread>
#include <vector>

static thread_local int device = 0;
static std::atomic<int> calls{0}, limit[4];
static hipError_t error = hipSuccess;
extern "C" hipError_t hipGetDevice(int *d) { *d = device; return hipSuccess; }
extern "C" hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int value) {
    ++calls;
    if (error != hipSuccess) return error;
    limit[device % 4] = value;
    return hipSuccess;
}
static ojx::DynLds lds;
static hipError_t raise(int d, size_t bytes) { device = d; return ojx::raise_dyn_lds(&lds, bytes, &lds); }
#define CHECK(c) if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; }
int main() {
    CHECK(raise(0, 100000) == hipSuccess && limit[0] == 100000 && calls == 1)
    CHECK(raise(0, 90000) == hipSuccess && raise(0, 100000) == hipSuccess && calls == 1)
    CHECK(raise(1, 90000) == hipSuccess && limit[1] == 90000 && calls == 2)       // a device of its own
    CHECK(raise(0, 120000) == hipSuccess && limit[0] == 120000 && limit[1] == 90000)
    error = hipErrorInvalidValue;
    CHECK(raise(2, 130000) == hipErrorInvalidValue)                                // handed on, nothing kept
    error = hipSuccess;
    CHECK(raise(2, 80000) == hipSuccess && limit[2] == 80000)
    calls = 0;
    CHECK(raise(ojx::DynLds::kDevices + 3, 70000) == hipSuccess && raise(ojx::DynLds::kDevices + 3, 70000) == hipSuccess)
    CHECK(calls == 2)                                                              // not kept: every call
    limit[3] = 0;
    std::vector<std::thread> t;
    for (int i = 0; i < 8; ++i)
        t.emplace_back([i] { for (int k = 0; k < 200; ++k) raise(3, 66000 + 8 * ((i * 37 + k * 11) % 500)); });
    for (auto &x : t) x.join();
    CHECK(limit[3] >= 66000 && limit[3] == (int)lds.granted[3].load())
    std::printf("OK\n");
}
"""


def test_limits_by_device(tmp_path):
    src, exe = tmp_path / "lds.cpp", tmp_path / "lds"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROCM, "include"), "-I",
                    os.path.join(ROOT, "ojasx-vector-24x96_amd", "csrc"), str(src), "-o", str(exe), "-lpthread"],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout


def test_every_limit_goes_through_it():
    """No other call sets a kernel's limit, kept for the process alone."""
    csrc = os.path.join(ROOT, "ojasx-vector-24x96_amd", "csrc")
    for name in os.listdir(csrc):
        if name != "dyn_lds.h":
            with open(os.path.join(csrc, name)) as f:
                assert "hipFuncSetAttribute(" not in f.read(), name
