/* Where a running sum over the bins of the sampler's histogram reaches a goal.
 * Plain C++, for the kernel and for a test on the host. */
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define SM100_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define SM100_HOST_DEVICE inline
#endif

namespace sm100 {

/* Sums of bins are whole numbers (ids, or estimated weight in units of 2^-40):
 * they do not depend on the order in which threads and CTAs add them up, so what
 * a thread takes as the sum before its first bin is what its neighbour has after
 * its last one.  With f32 sums the two differ in the last places: a goal between
 * them has two owners, whose writes then race, or none. */
typedef uint64_t BinSum;

/* Whether a sum that goes from `was` to `now` in a bin with ids reaches the goal
 * there; `first`: no id lies before the bin (a goal of nothing is reached in the
 * first bin with ids).  Of all bins with ids one answers yes, or none where the
 * whole sum is below the goal. */
template <typename Sum>
SM100_HOST_DEVICE bool reaches(Sum was, Sum now, bool first, Sum goal) {
  return now >= goal && (was < goal || first);
}

}  // namespace sm100
