// kvq_ring.h — the bookkeeping of a warp's ring of page copies: plain C++, so
// that the host can run it too.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define KVQ_RING_FN __host__ __device__ __forceinline__
#else
#define KVQ_RING_FN inline
#endif

namespace bitnet {

// Stages are filled and used in turn.  A full ring and an empty one have their
// next stages alike, so the copies in flight are counted by themselves: before
// its shared memory may go, a warp waits for each of them (wait for `take` with
// `parity`, then used(), until flying is 0).
template <int STAGES>
struct StageRing {
  int fill = 0, take = 0;  // stages, the next to fetch into and the next to use
  int flying = 0;          // stages fetched into and not yet used
  uint32_t parity = 0;     // of the copies that `take` waits for
  KVQ_RING_FN void fetched() {
    fill = fill + 1 == STAGES ? 0 : fill + 1;
    ++flying;
  }
  KVQ_RING_FN void used() {
    --flying;
    if (++take == STAGES) {
      take = 0;
      parity ^= 1;
    }
  }
};

}  // namespace bitnet
