// Places in a ring of buffers whose barriers change parity every round, and which rounds of them
// hold loads that have been issued: what a kernel that gives up has to wait for.  Host code too, so
// that the bookkeeping can be tested without a GPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define FG_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FG_HOST_DEVICE inline
#endif

namespace fg {

// A place in a ring of `n` slots or buffers and the parity of its current round.
struct Place {
  uint32_t at = 0, parity = 0;
  FG_HOST_DEVICE void next(uint32_t n) {
    if (++at == n) {
      at = 0;
      parity ^= 1;
    }
  }
};

// The parity of the last load into slot `k`, with `next` the place of the next load: the slots from
// there on belong to the round before.
FG_HOST_DEVICE uint32_t last_round(const Place& next, uint32_t k) {
  return k < next.at ? next.parity : next.parity ^ 1;
}

// Loads through one barrier, one after the other.
struct Loads {
  uint32_t issued = 0;
  FG_HOST_DEVICE bool any() const { return issued > 0; }
  FG_HOST_DEVICE uint32_t last_parity() const { return (issued - 1) & 1; }
};

}  // namespace fg
