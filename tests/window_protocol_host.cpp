// The host-side build of the kernels' plain arithmetic, for tests through ctypes.
#include "bounded_wait.h"
#include "window_turns.h"

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

int turns_size() {
    return (int) sizeof(cubk::WindowTurns);
}

void turns_reset(cubk::WindowTurns *t) {
    t->reset();
}

void turns_add(cubk::WindowTurns *t, int turn, int item) {
    t->add(turn, item);
}

void turns_gave_up(cubk::WindowTurns *t, int turn) {   // atomicMin on the device
    t->first_bad = turn < t->first_bad ? turn : t->first_bad;
}

int turns_first_bad(const cubk::WindowTurns *t) {
    return t->first_bad;
}

int turns_known(const cubk::WindowTurns *t) {
    return t->known;
}

int turns_item(const cubk::WindowTurns *t, int turn) {
    return t->item(turn);
}

}
