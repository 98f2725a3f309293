// Places in rings of shared-memory stages, as the producers and the consumers
// of the 4-bit head count them (plain integers: they hold on the host too).
#pragma once
#include <cstdint>

namespace mstar {

// A place in a ring of `n` stages and the parity of its current use.
struct Ring {
  uint32_t i = 0, parity = 0;
  __host__ __device__ __forceinline__ void next(uint32_t n) {
    if (++i == n) i = 0, parity ^= 1u;
  }
};

// A ring for each of LANES consumers, of every LANES-th stage of `stages` (a
// multiple of LANES).  A wait by parity sees one phase: it passes too early for a
// consumer that has not seen the phase before end.  So a stage never changes
// lanes: each of its phases is waited for by the same consumers, and they give it
// back before it is filled again, however many blocks either lane has.
template <int LANES>
struct LaneRings {
  Ring ring[LANES];
  __host__ __device__ __forceinline__ uint32_t stage(int lane) const {
    return ring[lane].i * (uint32_t)LANES + (uint32_t)lane;
  }
  __host__ __device__ __forceinline__ uint32_t parity(int lane) const { return ring[lane].parity; }
  __host__ __device__ __forceinline__ void next(int lane, uint32_t stages) { ring[lane].next(stages / LANES); }
};

}  // namespace mstar
