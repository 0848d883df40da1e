// phases.cuh -- which phase of which barrier the steps of a pipeline wait for.  Plain
// arithmetic, the same on the host, where tests/test_phases.py runs it.
#pragma once

#include <stdint.h>

namespace tbk {

// A ring of STAGES barriers: step j uses barrier j % STAGES, each use one completion.
template <int STAGES>
struct Ring {
    static constexpr int stage(int j) { return j % STAGES; }
    static constexpr uint32_t parity(int j) { return (uint32_t)(j / STAGES) & 1u; }
    // Whether step j takes a stage that an earlier step, j - STAGES, has to free.
    static constexpr bool reused(int j) { return j >= STAGES; }
    // Whether a later step of `steps` waits for step j's stage to be free.  A completion
    // that nobody waits for may come after the block has ended, when its shared memory
    // is another's.
    static constexpr bool awaited(int j, int steps) { return j + STAGES < steps; }
};

// The phases of up to 32 barriers that are waited for when there is something to wait
// for, a bit each: the one that the next completion of barrier i ends.  A wait that gives
// up leaves the phase as it is, so that a second one asks for the same completion; past it
// the barrier would answer for the phase before, at once, with the copy still in flight.
struct Phases {
    uint32_t bits = 0;
    // came(parity): the bounded wait of barrier i
    template <typename F>
    __device__ __forceinline__ bool wait(int i, F came) {
        if (!came(bits >> i & 1u)) return false;
        bits ^= 1u << i;
        return true;
    }
};

}  // namespace tbk
