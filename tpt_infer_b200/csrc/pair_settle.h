// pair_settle.h -- how an aborting SM pair closes the stages that only one of its
// two producers issued. Plain C++ as well, so that the rule is tested without a GPU.
//
// Stage i of the pair counts on the leader's full barrier: one arrival, the
// leader's, which expects the bytes of both CTAs' copies, and those bytes as the
// copies land. `mine` and `theirs` are the stages that the leader's and the other
// CTA's producer issued. A stage that both issued completes by itself. One that only
// the leader issued lacks the other's bytes: they are counted as if they had landed.
// One that only the other CTA issued lacks the arrival: it is made, expecting that
// CTA's bytes alone. Each phase then ends when the copies that are in flight have
// landed, and not before.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define PAIR_SETTLE_FN __host__ __device__ __forceinline__
#else
#define PAIR_SETTLE_FN inline
#endif

namespace tpt {

struct PairSettle {
    int arrive;         // 1: an arrival that expects `expect` bytes is missing
    uint32_t expect;
    uint32_t complete;  // bytes to count as landed
};

// stage i < max(mine, theirs), `bytes` of each CTA
PAIR_SETTLE_FN PairSettle pair_settle(int i, int mine, int theirs, uint32_t bytes) {
    PairSettle p = {0, 0, 0};
    if (i >= mine) {
        p.arrive = 1;
        p.expect = bytes;
    } else if (i >= theirs) {
        p.complete = bytes;
    }
    return p;
}

}  // namespace tpt
