"""The launches' host side and order, without a GPU."""
import os
import re
import subprocess

import pytest
import torch

from libnrn_b200 import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "libnrn_b200", "csrc")


ALLOW = r"""
// Two threads allow one kernel different sizes; the runtime's call of the smaller takes its time.
#include <cuda_runtime.h>
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>

static cudaError_t set_attribute(int bytes);
template <typename K>
cudaError_t fake_attribute(K*, cudaFuncAttribute, int bytes) { return set_attribute(bytes); }
#define cudaFuncSetAttribute fake_attribute
#include "launch.h"

static std::mutex m;
static std::condition_variable changed;
static bool small_in, large_done;
static int attribute;

namespace nrn { int sm_count_current() { return 1; } }
extern "C" cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
static cudaError_t set_attribute(int bytes) {
    std::unique_lock<std::mutex> l(m);
    if (bytes == 100) {
        small_in = true;
        changed.notify_all();
        changed.wait_for(l, std::chrono::milliseconds(300), [] { return large_done; });   // lets the other overtake, if it can
    }
    attribute = bytes;
    if (bytes == 200) {
        large_done = true;
        changed.notify_all();
    }
    return cudaSuccess;
}

void kernel() {}

int main() {
    std::thread a([] { nrn::allow_shared<kernel>(100); });
    std::thread b([] {
        std::unique_lock<std::mutex> l(m);
        changed.wait(l, [] { return small_in; });
        l.unlock();
        nrn::allow_shared<kernel>(200);
    });
    a.join();
    b.join();
    if (attribute != 200) return printf("left at %d bytes\n", attribute), 1;
    nrn::allow_shared<kernel>(150);
    if (attribute != 200) return printf("lowered to %d bytes\n", attribute), 1;
    return 0;
}
"""


def test_shared_memory_is_only_raised(tmp_path):
    src, exe = tmp_path / "allow.cpp", tmp_path / "allow"
    src.write_text(ALLOW)
    from libnrn_b200 import build as B
    r = subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-pthread", f"-I{CSRC}", f"-I{os.path.join(ROOT, 'include')}", "-I/usr/local/cuda/include",
                        f"-I{os.path.join(B.NCCL, 'include')}", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    for _ in range(3):
        r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("name", ["linattn.cu", "scaled.cu", "gatednorm.cu"])
def test_no_kernel_lets_the_next_in_before_it_has_its_tmem(name):
    """tcgen05.alloc waits for columns without a limit: a block of the next kernel, on the same SM, could take them and wait
    for this one."""
    src = open(os.path.join(CSRC, name)).read()
    for kernel in re.split(r"\n(?=__global__)", src)[1:]:
        alloc = kernel.find("tcgen05.alloc")
        if alloc < 0:
            continue
        body = kernel[:alloc]
        for at in (m.start() for m in re.finditer(r"\blet_next\(\)", body)):
            # only where the block ends without any
            assert re.match(r"let_next\(\);\s*previous_done\(\);\s*return;", body[at:]), f"{name}: let_next before tcgen05.alloc"
        assert re.search(r"\blet_next\(\)", kernel[alloc:])


def test_a_stream_of_another_device_is_refused():
    from libnrn_b200._tensors import on

    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 0
    with pytest.raises(N.NrnError, match="stream"):
        with on(torch.device("cuda", 0), Stream()):
            pass
