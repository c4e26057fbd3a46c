// What a block of the tensor-memory window attention keeps about the items it works through, so that after a give-up every row
// without a result can be found. Plain arithmetic, so that it can be tested on the host.
#pragma once

#include "bounded_wait.h"

namespace cubk {

constexpr int kNoTurn = 0x7fffffff;

struct WindowTurns {
    // Four are enough. Turn T is begun before the queries of turn T - 2 are known to be used up, so that its warps may be as far back as
    // turn T - 3; an item is taken over (turn T + 1, not begun) only after that, when no warp can still give up in turn T - 3.
    int items[4];
    int known;       // turns begun or taken over
    int first_bad;   // the first turn in which a warp gave up before its rows

    CUBK_HOST_DEVICE void reset() {
        known = 0;
        first_bad = kNoTurn;
    }
    CUBK_HOST_DEVICE void add(int turn, int item) {
        items[turn & 3] = item;
        known = turn + 1;
    }
    CUBK_HOST_DEVICE int item(int turn) const {
        return items[turn & 3];
    }
};

}  // namespace cubk
