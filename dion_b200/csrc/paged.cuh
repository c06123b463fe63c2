// What the kernels around the paged cache share: how the cache and the new tokens are described, and the search for the
// sequence of a token.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dion {

// Largest b in [0, n) with offsets[b] <= row (0 if there is none), by a whole warp: 32 probes a round, so that up to 32
// sequences take one round of loads and up to 1024 two.  Any values of `offsets` keep the result in range.
__device__ __forceinline__ int sequence_of(const int* __restrict__ offsets, int n, int row, int lane) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && (lane == 0 || offsets[at] <= row));
    const int last = below == 0xffffffffu ? 31 : __ffs(~below) - 2;  // of the unbroken run from lane 0
    lo += last * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

__device__ __forceinline__ void bad_argument(int* status) { atomicCAS(status, 0, 5 /* kStatusBadArgument */); }

}  // namespace dion
