// The count of copies that a producer issues into two slots in turn, copy j
// into slot j & 1 as that slot's phase j >> 1. A copy gets its slot by being
// counted, so that whoever leaves the producer's loop early still finds every
// copy that may be in flight in [oldest(), issued()). Plain C++: the tests
// compile it for the host.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define B2_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define B2_HOST_DEVICE inline
#endif

namespace b2 {

class SlotPair {
    uint32_t n = 0;

  public:
    B2_HOST_DEVICE static uint32_t slot(uint32_t copy) { return copy & 1u; }
    B2_HOST_DEVICE static uint32_t parity(uint32_t copy) { return (copy >> 1) & 1u; }
    B2_HOST_DEVICE uint32_t issued() const { return n; }
    // The slot of the next copy, and whether (and for which parity) it has to be given back before.
    B2_HOST_DEVICE uint32_t next() const { return slot(n); }
    B2_HOST_DEVICE bool in_use() const { return n >= 2; }
    B2_HOST_DEVICE uint32_t free_parity() const { return parity(n - 2); }
    // The oldest copy that may be in flight: those before it gave their slots back.
    B2_HOST_DEVICE uint32_t oldest() const { return n > 2 ? n - 2 : 0; }
    // Counts the next copy, which is issued right behind; its slot. withdraw() where it was not issued after
    // all: a count too high costs a bounded wait, one too low leaves a copy in flight.
    B2_HOST_DEVICE uint32_t begin() { return slot(n++); }
    B2_HOST_DEVICE void withdraw() { --n; }
};

}  // namespace b2
