// The counter-based random numbers of the kernels that choose tokens: the number of a (seed, index of the token being produced).
#pragma once

#include "common.cuh"

namespace mlr {

__device__ __forceinline__ float uniform_from_seed(unsigned long long seed, long long index) {
  unsigned long long z = seed + (unsigned long long)(index + 1) * 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  z = z ^ (z >> 31);
  return (float)(z >> 40) * (1.0f / 16777216.0f);
}

}  // namespace mlr
