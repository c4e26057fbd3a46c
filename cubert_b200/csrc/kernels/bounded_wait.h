// When a bounded wait on the device is over. Plain arithmetic, so that it can be tested on the host.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define CUBK_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define CUBK_HOST_DEVICE inline
#endif

namespace cubk {

constexpr uint32_t kBarrierWaitNs = 200u * 1000 * 1000;   // 0.2 s: five orders above a copy's latency
constexpr uint32_t kBarrierGapNs = 1000u * 1000;          // counted at most between two readings of the clock

// Adds up the time between readings (the clock's low 32 bits, in nanoseconds). A block that was taken off its SM comes back after any
// length of time without having polled, so a gap counts as a millisecond at most: what is waited for gets its 0.2 s while the block runs.
struct WaitClock {
    uint32_t last = 0, waited = 0;

    CUBK_HOST_DEVICE bool over(uint32_t now) {
        const uint32_t gap = last != 0 ? now - last : 0;
        waited += gap < kBarrierGapNs ? gap : kBarrierGapNs;
        last = now;
        return waited > kBarrierWaitNs;
    }
};

}  // namespace cubk
