"""What a launcher sets once a device (csrc/common.cuh), without a device: a program of the header, built here.  Two threads come at once, and a
setting fails."""
import subprocess

PROGRAM = r"""
#include "common.cuh"
#include <chrono>
#include <cstdio>
#include <thread>
int main() {
    using std::this_thread::sleep_for;
    using std::chrono::milliseconds;
    // ---- the first thread is in the middle of its setting when the second comes: neither goes on before one setting is complete ----
    DeviceOnce once;
    std::atomic<int> begun{0}, complete{0}, early{0};
    auto launcher = [&](int ms) {
        if (once([&] { begun++; sleep_for(milliseconds(ms)); complete++; return cudaSuccess; }) != cudaSuccess || complete == 0) early++;
    };
    std::thread first(launcher, 400);
    while (begun == 0) sleep_for(milliseconds(1));
    std::thread second(launcher, 0);
    second.join();
    first.join();
    const int before = begun;
    launcher(0);                                            // set by now: not again
    printf("%d early, %d more\n", early.load(), begun.load() - before);
    // ---- a setting that fails is told to its caller, and tried again by the next ----
    DeviceOnce again;
    int calls = 0;
    const bool told = again([&] { ++calls; return cudaErrorInvalidValue; }) == cudaErrorInvalidValue;
    const bool mended = again([&] { ++calls; return cudaSuccess; }) == cudaSuccess && again([&] { ++calls; return cudaErrorInvalidValue; }) == cudaSuccess;
    printf("%d %d %d\n", told, mended, calls);
    return 0;
}
"""


def test_set_once(tmp_path):
    from tiny_inference_server_b200.kernels import build
    (tmp_path / "once.cu").write_text(PROGRAM)
    subprocess.run([build._nvcc(), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", build.CSRC, "-o", str(tmp_path / "once"), str(tmp_path / "once.cu")],
                   check=True)
    out = subprocess.run([str(tmp_path / "once")], check=True, capture_output=True, text=True, timeout=60).stdout
    assert out.split("\n")[:2] == ["0 early, 0 more", "1 1 2"], out
