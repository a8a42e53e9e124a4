// Waits that end, for barriers whose state is one bit (the parity of the phase that is not over yet).
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define FFCVB_EVERYWHERE __host__ __device__ __forceinline__
#else
#define FFCVB_EVERYWHERE inline
#endif

namespace ffcvb {

constexpr uint64_t kLongestWait = 2000000000ull; // ns
// What counts as waiting between two looks at the clock, at most: a longer time is one in which the whole block was not on the GPU.
constexpr uint64_t kLongestLook = 100000000ull;
constexpr uint32_t kTriesForALook = 64;

// One that waits for barriers' phases, one after another.  `gave_up` is all waiters' of a block: whoever waits longer than kLongestWait sets it, and no wait that has to try
// again lasts once it is set.  A waiter whose wait has run out waits no more: a later phase of that barrier has the parity that it waited for in vain, or the one
// before that, and would seem to be over.
struct Waiter {
    volatile int *gave_up;
    bool fine;
    FFCVB_EVERYWHERE explicit Waiter(volatile int *all) : gave_up(all), fine(true) {}
    // passed(): whether the phase is over; now(): nanoseconds.
    template <typename Passed, typename Now> FFCVB_EVERYWHERE bool operator()(Passed passed, Now now) {
        if (!fine) return false;
        if (passed()) return true;
        uint64_t last = 0, waited = 0;
        for (uint32_t tries = 1;; tries++) {
            if (passed()) return true;
            if (tries % kTriesForALook != 0) continue;
            if (*gave_up) return fine = false;
            const uint64_t time = now(), more = time - last;
            if (last != 0) waited += more < kLongestLook ? more : kLongestLook;
            last = time;
            if (waited > kLongestWait) {
                *gave_up = 1;
                return fine = false;
            }
        }
    }
};

} // namespace ffcvb
