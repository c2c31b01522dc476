// A ring of n slots that loads fill and products empty in turn, each slot with a barrier whose phases its loads complete. Plain
// arithmetic, so that it can be checked on the host.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define SRHPM_RING_FN __host__ __device__ __forceinline__
#else
#define SRHPM_RING_FN inline
#endif

namespace srhpm {

// the slot of load c (the c-th of all), and the parity of the phase that it completes
SRHPM_RING_FN uint32_t ring_slot(uint32_t c, uint32_t n) { return c % n; }
SRHPM_RING_FN uint32_t ring_parity(uint32_t c, uint32_t n) { return c / n & 1; }

// Loads that went out so far, of a warp that asks for n ahead and for one more behind each of `done` steps; idle: how many times it
// has asked since there were no more (negative: there are more). Loads done .. ring_issued - 1 may be in flight.
SRHPM_RING_FN uint32_t ring_issued(uint32_t done, uint32_t n, int idle) { return done + n - (uint32_t) (idle > 0 ? idle : 0); }

}  // namespace srhpm
