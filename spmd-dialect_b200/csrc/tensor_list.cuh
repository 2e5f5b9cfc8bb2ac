// tensor_list.cuh -- a list of tensors as work for one launch: the pieces all
// have one length, tensor k owns pieces first[k] .. first[k + 1), and a block
// finds the tensor of its piece by bisection.  The tables travel as kernel
// parameters, so a launch needs no upload and a captured launch keeps its own.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace spmdb200 {

// The last k with first[k] <= piece (first[0] = 0, ascending, `count` tensors
// of at least one piece each).
__device__ __forceinline__ int tensor_of(const int64_t *first, int count, int64_t piece) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= piece) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace spmdb200
