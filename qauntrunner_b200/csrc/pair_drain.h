// pair_drain.h -- how a pair of CTAs whose copies complete on barriers of the
// first one leaves when a wait gave up (fp8.cuh, fp4.cuh).  Host code too: the order of
// the steps is checked on the CPU.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define QRM_HD __host__ __device__ __forceinline__
#else
#define QRM_HD inline
#endif

namespace qrm {

// Waits until every copy that both CTAs have issued has landed.  mine, peer:
// stages that the first CTA and the other have issued, each one a copy of a
// share of the bytes that stage j's barrier (slot j % stages, phase j / stages)
// expects; the first CTA's issue is also the barrier's arrival.  A stage is
// issued only when the one `stages` before has landed in both, so the counts
// are at most `stages` apart and the last `stages` are all that can be in
// flight.
//   bars.expect(slot)    arrival, expecting the other CTA's share only
//   bars.complete(slot)  the other CTA's share, which will not come
//   bars.wait(slot, parity)
template <typename Bars>
QRM_HD void drain_pair(uint32_t mine, uint32_t peer, uint32_t stages, Bars& bars) {
    const uint32_t most = mine > peer ? mine : peer;
    for (uint32_t j = most > stages ? most - stages : 0; j < most; j++) {
        if (j >= mine) bars.expect(j % stages);
        else if (j >= peer) bars.complete(j % stages);
        bars.wait(j % stages, (j / stages) & 1u);
    }
}

}  // namespace qrm
