// The host-side build of the kernels' plain arithmetic, for tests through ctypes.
#include "bounded_wait.h"

extern "C" {

// Readings of the clock until a wait is over; n + 1 if none of the n readings ends it.
int wait_over_at(const uint64_t *readings, int n) {
    cubk::WaitClock clock;
    for (int i = 0; i < n; ++i) {
        if (clock.over((uint32_t) readings[i])) {
            return i + 1;
        }
    }
    return n + 1;
}

}
