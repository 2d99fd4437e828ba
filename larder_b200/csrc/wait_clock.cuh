// The clock of a bounded wait in one 32-bit register. Plain C++: also compiled without CUDA.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LB2_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define LB2_HOST_DEVICE inline
#endif

namespace lb2 {

// A wait's look at the clock: since is 0 at its first look, then what this returned; 1: more than limit_ns (up to 2^44) have
// passed. The stamp is the time in ticks of 2^16 ns (66 us), four to a tick and two more: never 0 or 1, whatever the tick, and
// two stamps' difference is the time between them, the wrap after 2^30 ticks (19 hours) among them.
LB2_HOST_DEVICE uint32_t wait_look(uint32_t since, uint64_t ns, uint64_t limit_ns) {
  const uint32_t now = uint32_t(ns >> 16) << 2 | 2u;
  if (since == 0) return now;
  return int32_t(now - since) > int32_t(limit_ns >> 16 << 2) ? 1u : since;
}

}  // namespace lb2
