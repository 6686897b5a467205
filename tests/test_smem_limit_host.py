"""What a kernel has been allowed of shared memory, by two host threads at once: csrc/smem_limit.h, compiled alone."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vectorsparse_b200", "csrc")

# A thread that asks for little is held up in the runtime's call, before it takes effect, until another that asks for much is through, or has been kept
# waiting for half a second.  What counts afterwards is the runtime's own state.
PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <future>
#include <thread>
#include "smem_limit.h"

int main() {
    vs::SmemLimit limit;
    std::atomic<int> runtime{0}, calls{0};
    std::promise<void> inside, large_done;
    auto done = large_done.get_future();
    std::thread small([&] {
        limit.raise(3, 60000, [&] {
            inside.set_value();
            done.wait_for(std::chrono::milliseconds(500));
            ++calls;
            runtime = 60000;
            return 0;
        });
    });
    inside.get_future().wait();
    std::thread large([&] {
        limit.raise(3, 130000, [&] { ++calls; runtime = 130000; return 0; });
        large_done.set_value();
    });
    small.join();
    large.join();
    auto set = [&](int bytes) { return [&, bytes] { ++calls; runtime = bytes; return 0; }; };
    limit.raise(3, 100000, set(100000));
    if (runtime != 130000 || calls != 2) return 1;                        // nothing taken back, nothing asked twice
    if (limit.raise(4, 1000, set(1000)) != 0 || calls != 3) return 2;     // another device
    if (limit.raise(4, 2000, [] { return 7; }) != 7) return 3;            // a refusal is passed on
    if (limit.raise(4, 2000, set(2000)) != 0 || runtime != 2000) return 4; // and asked for again
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_the_limit_only_grows(tmp_path):
    (tmp_path / "limit.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", CSRC, "-o", str(tmp_path / "limit"), str(tmp_path / "limit.cpp")], check=True)
    assert subprocess.run([str(tmp_path / "limit")], timeout=30).returncode == 0
