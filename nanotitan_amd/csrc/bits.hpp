// float32 to an activation type's bits by the hardware's conversion (nearest
// even): one instruction for two values, where the integer form of
// f32_to_bf16 takes six for one. Any NaN gives a NaN.
#pragma once

#include "common.hpp"

namespace nt {

template <typename T>
__device__ __forceinline__ typename elem<T>::storage to_bits(float f) {
  return elem<T>::store(f);
}
template <>
__device__ __forceinline__ uint16_t to_bits<bf16>(float f) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}

}  // namespace nt
