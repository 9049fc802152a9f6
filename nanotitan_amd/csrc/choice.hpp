// The order in which a router's choices are taken, for the layers of few tokens.
#pragma once

#include "common.hpp"

namespace nt {

// Choices in the order of nt_route_topk as one unsigned key, the larger first:
// the value's bits as an ordered integer (-0 as +0, every NaN below -inf), then
// the lower expert. 0: no choice.
__device__ __forceinline__ uint64_t choice_key(float z, int e) {
  uint32_t u = __float_as_uint(z);  // integers only: denormals keep their order
  if (u == 0x80000000u) u = 0u;
  const uint32_t ordered =
      (u & 0x7fffffffu) > 0x7f800000u ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
  return ((uint64_t)ordered << 32) | (uint32_t)~e;
}
__device__ __forceinline__ float choice_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u == 0u ? 0x7fc00000u : (u >> 31) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int choice_expert(uint64_t key) { return (int)~(uint32_t)key; }

}  // namespace nt
