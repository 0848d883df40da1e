"""The barrier arithmetic of the pipelined kernels (csrc/phases.cuh), on the host: a
small C++ program runs it against barriers that count their phases."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tensorbit-run_b200", "csrc")

FAKE = """
#include <cassert>
#include <cstdio>
#include "phases.cuh"
// A barrier of one arrival a phase, and its wait: whether phase `parity` is complete.
struct Barrier {
    int completed = 0, awaited = 0;
    void complete() { ++completed; }
    bool done(uint32_t parity) const { return (uint32_t)(completed & 1) != parity; }
    bool wait(uint32_t parity) { return done(parity) ? (awaited = completed, true) : false; }
};
"""


@pytest.fixture
def run(tmp_path):
    def go(body):
        src, exe = tmp_path / "t.cpp", tmp_path / "t"
        src.write_text(FAKE + body)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-D__device__=",
                        "-D__host__=", "-D__forceinline__=inline", "-I", CSRC, str(src), "-o",
                        str(exe)], check=True, timeout=120)
        subprocess.run([str(exe)], check=True, timeout=60)
    return go


def test_no_stage_is_freed_for_nobody(run):
    """A producer that fills a ring, and a consumer that frees each stage when a later
    step waits for it: each wait is for the phase that the step before completed, and
    at the end every completion has been waited for."""
    run("""
template <int S> void ring(int steps) {
    using R = tbk::Ring<S>;
    Barrier full[S], free[S];
    for (int j = 0; j < steps; ++j) {
        Barrier& f = free[R::stage(j)];
        if (R::reused(j)) {
            assert(f.completed == j / S);  // once by each earlier use
            assert(f.wait(R::parity(j - S)) && !f.done(R::parity(j)));
        }
        Barrier& b = full[R::stage(j)];
        assert(!b.done(R::parity(j)));
        b.complete();
        assert(b.wait(R::parity(j)));
        if (R::awaited(j, steps)) f.complete();
    }
    for (int i = 0; i < S; ++i) {
        assert(free[i].awaited == free[i].completed);
        assert(full[i].awaited == full[i].completed);
    }
}
int main() {
    for (int steps = 0; steps < 20; ++steps) ring<1>(steps), ring<2>(steps), ring<3>(steps);
}
""")


def test_a_wait_that_gave_up_asks_again(run):
    """A copy that comes after its wait gave up: the clean-up's wait is for that copy,
    not for the one before, at either parity."""
    run("""
int main() {
    for (int before = 0; before < 5; ++before) {
        Barrier b[2];
        tbk::Phases p;
        auto came = [&](int i) { return p.wait(i, [&](uint32_t parity) { return b[i].wait(parity); }); };
        for (int j = 0; j < before; ++j) {
            b[1].complete();
            assert(came(1));
            assert(!came(1));  // one wait a completion
        }
        assert(!came(1) && !came(1));  // in flight
        assert(!came(0));
        b[1].complete();
        assert(came(1) && !came(0));
        b[0].complete();
        assert(came(0) && !came(1));
    }
}
""")


def test_a_lost_copy_leaves_none_in_flight(run):
    """A ring of stages filled ahead, where the copies from step `late` on come only
    after a wait gave up on them: waiting for that step's stage again and for those
    behind it, those of steps without a copy left out, brings all of them in."""
    run("""
template <int S> void ring(int steps, int late, unsigned missing) {
    Barrier b[S];
    int asked[S] = {}, in_flight = 0;
    tbk::Phases p;
    auto has = [&](int n) { return n < steps && !(missing >> n & 1); };
    auto issue = [&](int n) {
        if (!has(n)) return;
        if (n >= late) asked[n % S] = 1, ++in_flight; else b[n % S].complete();
    };
    auto came = [&](int i) {
        return p.wait(i, [&](uint32_t parity) {
            if (b[i].wait(parity)) return true;
            if (asked[i] == 1) { asked[i] = 2; return false; }      // gives up
            if (asked[i] == 2) { b[i].complete(); --in_flight; }    // late, but there
            return b[i].wait(parity);
        });
    };
    for (int n = 0; n < S - 1; ++n) issue(n);
    for (int n = 0; n < steps; ++n) {
        issue(n + S - 1);
        if (!has(n) || came(n % S)) continue;
        for (int i = 0; i < S; ++i)
            if (has(n + i) && !came((n + i) % S)) came((n + i) % S);
        assert(in_flight == 0);
        return;
    }
    assert(in_flight == 0);
}
int main() {
    for (int steps = 0; steps < 12; ++steps)
        for (int late = 0; late <= steps; ++late)
            for (unsigned missing = 0; missing < 4096; missing += 37)
                ring<2>(steps, late, missing), ring<3>(steps, late, missing);
}
""")
