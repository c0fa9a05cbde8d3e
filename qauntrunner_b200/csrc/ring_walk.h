// ring_walk.h -- how a CTA's threads walk its rows through a ring of copies in
// shared memory (norm.cuh), and what becomes of the ring when a wait for a copy
// gave up.  Host code too: the order of the steps is checked on the CPU.
#pragma once
#include <stdint.h>

#ifndef QRM_HD
#ifdef __CUDACC__
#define QRM_HD __host__ __device__ __forceinline__
#else
#define QRM_HD inline
#endif
#endif

namespace qrm {

// A CTA's rows are number 0, 1, ... `count` - 1; slot n % slots takes row n.  The
// lead thread issues the copies, the first `slots` of them ahead.  For each row
// every thread calls ring_wait, reads the row from its slot, meets the others at a
// barrier and calls ring_next with the row that is `slots` on.
//
// A thread whose wait gave up says so (ring.fail) and goes on with what the slot
// holds: what the CTA writes is spoilt, and whoever walks the ring has to make it
// show at the end (ring.failed).  From the next barrier on no slot is loaded again,
// so no two copies are ever on their way to one slot.  At the end the lead calls
// ring_drain, so that none lands behind the CTA's.
//   ring.i, ring.parity            the row's slot and its phase
//   ring.slots
//   ring.wait(slot, parity)        false: it gave up (at once where another one has)
//   ring.drain(slot, parity)       the same, but for its own time
//   ring.lead()
//   ring.load(slot, n)             row n, if there is one
//   ring.fail(), ring.failed()
//   ring.stop(n)                   row n was the first not to be loaded (said again for later ones)
template <typename Ring>
QRM_HD void ring_wait(Ring& ring) {
    if (!ring.wait(ring.i, ring.parity)) ring.fail();
}
template <typename Ring, typename Row>
QRM_HD void ring_next(Ring& ring, Row ahead) {
    if (ring.lead()) {
        if (!ring.failed()) ring.load(ring.i, ahead);
        else ring.stop(ahead);
    }
    if (++ring.i == ring.slots) {
        ring.i = 0;
        ring.parity ^= 1;
    }
}
// the copies that may be on their way when `issued` rows were loaded
template <typename Ring>
QRM_HD void ring_drain(Ring& ring, uint32_t issued) {
    for (uint32_t n = issued > ring.slots ? issued - ring.slots : 0; n < issued; n++) ring.drain(n % ring.slots, n / ring.slots & 1);
}

}  // namespace qrm
