// shared_stages.h -- the stages in shared memory of k_shared_tc.cu, which a step's keys and values
// are copied to. (Host and device: the order of waits that follows is walked through on the CPU,
// tests/shared_stages_check.cpp.)
//
// Steps are counted through all items of a CTA. Step n lies in stage n % N, and the barrier of
// that stage completes its phase n / N when the MMAs have read all of it: P V of a step is issued
// behind its S, so that is when its O is computed. Rows of step n are copied when step n - N is read.
// A wait tells phases apart by their parity, so it has to come before the barrier is two phases further.
// The phase after the one that a copy waits for is completed by the step that is copied, so
// it cannot be passed. (With one barrier for all steps it could be: S of a step is computed before
// P V of the step before it, so a loader may be a step ahead of the barrier, or behind it.)
#pragma once

#include <cstdint>

namespace tie {

template <uint32_t N>
struct Stages {
    static constexpr uint32_t of(uint32_t step) { return step % N; }
    static constexpr uint32_t phase(uint32_t step) { return step / N; }
    // its stage holds another step's rows, and which one's
    static constexpr bool used(uint32_t step) { return step >= N; }
    static constexpr uint32_t before(uint32_t step) { return step - N; }
};

}  // namespace tie
