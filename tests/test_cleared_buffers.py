"""A context's counters (csrc/sq8_buffers.h, reserve_cleared) on the CPU, against a stand-in for the runtime: no call may be
handed counters that were never cleared."""
import os
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "siliconed_amd", "csrc")
PROBE = r"""
#include "sq8_buffers.h"
#include <assert.h>
#include <set>
#include <stdio.h>
#include <stdlib.h>
static std::set<void *> live;
static bool captured = false;
extern "C" {
hipError_t hipMalloc(void **p, size_t bytes) { live.insert(*p = malloc(bytes)); return hipSuccess; }
hipError_t hipFree(void *p) { assert(live.erase(p) == 1); free(p); return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
    *s = captured ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipGetLastError(void) { return hipSuccess; }
}
int main() {
    sq8::Buffer b{};
    sq8::SetAside *aside = nullptr;
    hipError_t answer = hipErrorLaunchFailure;
    void *cleared = nullptr;
    size_t cleared_bytes = 0;
    auto reserve = [&](size_t bytes) {
        return sq8::reserve_cleared(b, bytes, 64, nullptr, aside, [&](void *at, size_t n) {
            if (answer == hipSuccess) cleared = at, cleared_bytes = n;
            return answer;
        });
    };
    for (int i = 0; i < 2; ++i) assert(reserve(16) == hipErrorLaunchFailure && !b.at && !b.bytes && live.empty());  // not kept
    answer = hipSuccess;
    assert(reserve(16) == hipSuccess && b.bytes == 64 && cleared == b.at && cleared_bytes == 64);
    cleared = nullptr;
    assert(reserve(64) == hipSuccess && !cleared);                              // clean: as every call leaves it
    captured = true;
    assert(reserve(65) == hipErrorStreamCaptureUnsupported && b.bytes == 64 && !b.in_graph);
    assert(reserve(32) == hipSuccess && b.in_graph && !cleared);
    void *graphs = b.at;
    captured = false;
    answer = hipErrorLaunchFailure;
    assert(reserve(1000) == hipErrorLaunchFailure && !b.at && live.size() == 1 && live.count(graphs));
    answer = hipSuccess;
    assert(reserve(100) == hipSuccess && cleared == b.at && cleared_bytes == 100 && !b.in_graph);
    sq8::release(b);
    sq8::release(aside);
    assert(live.empty());
    puts("ok");
}
"""


def test_counters_that_were_not_cleared_are_given_back(tmp_path):
    src, exe = str(tmp_path / "probe.cpp"), str(tmp_path / "probe")
    with open(src, "w") as f:
        f.write(PROBE)
    r = subprocess.run(["g++", "-std=c++17", "-g", "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include", "-I", CSRC, src, "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stderr
