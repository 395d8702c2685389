"""How the kernels' waits end (csrc/tq_wait.h), compiled for the host with a scripted barrier and clock."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "leankv_b200", "csrc")

PROGRAM = r"""
#include "tq_wait.h"
#include <cstdio>

int main() {
    uint64_t clock = 0;
    int tries = 0, ready_at = 0;
    const auto now = [&] { return clock; };
    const auto attempt = [&] { clock += 10000; return ++tries >= ready_at; };   // 10 us each
    volatile int failed = 0;
    const auto start = [&](int ready, int f) { clock = 5; tries = 0; ready_at = ready; failed = f; };
#define CHECK(x) if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; }
    // work that comes
    start(1, 0);
    CHECK(tq::wait_turn(attempt, now, &failed) && tries == 1 && failed == 0);
    start(500, 0);
    CHECK(tq::wait_turn(attempt, now, &failed) && tries == 500 && failed == 0);
    // another wait ran out: given up at once
    start(500, 1);
    CHECK(!tq::wait_turn(attempt, now, &failed) && tries == 1);
    // work that never comes: given up after the limit, and the others learn of it
    start(1 << 30, 0);
    CHECK(!tq::wait_turn(attempt, now, &failed) && failed == 1);
    CHECK(clock > tq::WAIT_NS && clock < tq::WAIT_NS + 100000);
    // issued work is waited for although another wait ran out, so that its memory is not taken away under it
    start(500, 1);
    CHECK(tq::wait_issued(attempt, now) && tries == 500);
    // ... and not for ever
    start(1 << 30, 1);
    CHECK(!tq::wait_issued(attempt, now));
    CHECK(clock > tq::WAIT_NS && clock < tq::WAIT_NS + 100000);
    return 0;
}
"""


def test_waits_end(tmp_path):
    src, exe = tmp_path / "wait.cpp", tmp_path / "wait"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_prompt_kernel_waits_for_issued_products_before_it_reuses_their_memory():
    """The barrier of all products is waited for by the wait that a failure elsewhere does not cut short."""
    with open(os.path.join(CSRC, "tq_attn_q8_prompt.cu")) as f:
        source = f.read()
    assert "mbar_wait_issued(done, 0)" in source and "mbar_wait(done" not in source
