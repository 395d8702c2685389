// tq_wait.h — how long a kernel waits on a barrier, apart from the barrier itself (host code compiles it too).
//
// attempt() asks once whether the barrier's phase has ended (and may suspend the thread for some microseconds), now()
// is a clock in nanoseconds.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define TQ_WAIT_FN __device__ __forceinline__
#else
#define TQ_WAIT_FN inline
#endif

namespace tq {

constexpr uint64_t WAIT_NS = 1000000000ull;

// Waits for work that another part of the CTA may never do: false once a wait of the CTA has run out, this one
// (which raises *failed) or any other.
template <typename Attempt, typename Now>
TQ_WAIT_FN bool wait_turn(Attempt attempt, Now now, volatile int* failed) {
    const uint64_t until = now() + WAIT_NS;
    while (!attempt()) {
        if (*failed) return false;
        if (now() > until) {
            *failed = 1;
            return false;
        }
    }
    return true;
}

// Waits for what has been issued and is under way (a copy, a product), whether or not another wait has run out: its
// memory must stay as it is until then.  False if it did not end within the limit.
template <typename Attempt, typename Now>
TQ_WAIT_FN bool wait_issued(Attempt attempt, Now now) {
    const uint64_t until = now() + WAIT_NS;
    while (!attempt())
        if (now() > until) return false;
    return true;
}

}  // namespace tq
