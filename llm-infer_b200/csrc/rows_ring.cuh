// The order in which a ring of whole rows in shared memory is filled, waited for and left, apart from the device's instructions so that it
// can be followed without one.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define B200_RING_FN __device__ __forceinline__
#else
#define B200_RING_FN inline
#endif

namespace b200 {

// Rows 0 .. mine - 1 through SLOTS slots. Row n lies in slot n % SLOTS, whose barrier completes a phase per row.
//   ask(n, slot)            requests row n; the slot is free
//   wait(slot, phase)       whether the row has arrived; false once the wait's limit ran out
//   reduce(n, slot, there)  reads row n; false, in every thread alike, where the wait of one of them ran out. Behind it the slot is read
//   finish(n)               what is left of row n
//   lose(n)                 rows n and further are given up: nothing is requested any more, and what was requested has been waited
//                           for once more, so that no copy writes a slot that is gone
template <uint32_t SLOTS, class Ask, class Wait, class Reduce, class Finish, class Lose>
B200_RING_FN void run_ring(uint32_t mine, Ask ask, Wait wait, Reduce reduce, Finish finish, Lose lose) {
    for (uint32_t n = 0; n < SLOTS && n < mine; ++n) ask(n, n);
    uint32_t slot = 0, phase = 0;
    for (uint32_t n = 0; n < mine; ++n) {
        if (!reduce(n, slot, wait(slot, phase))) {
            for (uint32_t i = 0; i < SLOTS && n + i < mine; ++i) {
                wait(slot, phase);
                if (++slot == SLOTS) slot = 0, phase ^= 1;
            }
            lose(n);
            return;
        }
        if (n + SLOTS < mine) ask(n + SLOTS, slot);
        finish(n);
        if (++slot == SLOTS) slot = 0, phase ^= 1;
    }
}

}  // namespace b200
