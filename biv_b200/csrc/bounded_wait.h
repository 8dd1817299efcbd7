// The bounded wait of the expert kernels' roles for one another.  Plain C++, without the CUDA
// headers, so that the rule can be tested where there is no GPU.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define BIV_WAIT_FN __device__ __forceinline__
#else
#define BIV_WAIT_FN inline
#endif

namespace bivmoe {

constexpr uint64_t kWaitNs = 2000000000ull;

// Waits until ready; false when it gave up.
//   w.ready()   one try           w.pause()   between two tries
//   w.late(k)   the k-th look, once in EVERY tries, at whether to give up
template <int EVERY, class W>
BIV_WAIT_FN bool bounded_wait(W w) {
    for (uint32_t i = 1; !w.ready(); i++) {
        if (i % EVERY == 0 && w.late(i / EVERY)) return false;
        w.pause();
    }
    return true;
}

// The same for the lanes of a warp, which go on, or leave, together: w.all(v) whether v holds for all
// of them.  A lane that sees another role's flag one turn before the others would by itself leave for
// the end of the kernel, and they would go on without it to what a whole warp has to execute
// (tensor-memory loads and stores, matrix instructions, shuffles).
template <int EVERY, class W>
BIV_WAIT_FN bool bounded_wait_together(W w) {
    const bool here = bounded_wait<EVERY>(w);
    return w.all(here);
}

// When a wait that looks at the clock gives up: kWaitNs after its first look, or after the last one at
// which another role was at something that its own work bounds, however long that takes.
struct WaitClock {
    uint64_t t0 = 0;
    BIV_WAIT_FN bool late(uint32_t look, uint64_t now_ns, bool at_work) {
        if (look == 1 || at_work) t0 = now_ns;
        return now_ns - t0 >= kWaitNs;
    }
};

// The last fills of a copying warp that may be under way yet.  It fills every STEP-th place of a line that goes
// round a ring of SLOTS, and a slot again only after its fill before has landed and been used: so the last
// SLOTS / STEP fills at most.  wait(slot, parity) of each, the oldest first; `last` is the place of the last one,
// `fills` how many there were.
template <int SLOTS, int STEP, class F>
BIV_WAIT_FN void wait_for_last_fills(uint32_t last, uint32_t fills, F wait) {
    static_assert(SLOTS % STEP == 0, "a warp's slots are its own");
    for (uint32_t i = fills < SLOTS / STEP ? fills : SLOTS / STEP; i--;) {
        const uint32_t at = last - STEP * i;
        wait(at % SLOTS, (at / SLOTS) & 1);
    }
}

// What a warp does that gave up on a wait while others may meet at a barrier that counts it: it arrives
// there for them (m.arrive()) until all have left (m.all_left()), each at its next wait; `turns` bounds
// that.  An arrival too many only ends a meeting early, which spoils nothing but results that the
// status disowns.  (Meetings at mbarriers, which a bounded wait could leave, cost the kernels 1 to 5 %.)
template <class M>
BIV_WAIT_FN void arrive_until_all_left(M m, uint32_t turns) {
    for (uint32_t i = 0; i < turns && !m.all_left(); i++) m.arrive();
}

}  // namespace bivmoe
