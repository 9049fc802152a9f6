// What the int8 products share: their arguments, the experts' rows and the
// epilogues. Tiles of many rows: int8_gemm.hip; few rows: int8_few.hip.
#pragma once

#include <type_traits>

#include "bits.hpp"
#include "gelu.hpp"
#include "int8.hpp"

namespace nt {

enum Int8Epilogue {
  kInt8Plain = NT_INT8_PLAIN,
  kInt8SwiGLU = NT_INT8_SWIGLU,
  kInt8Gelu = NT_INT8_GELU
};

struct Int8Gemm {
  const int8_t* x;          // rows of integers, and their scales [A]
  const float* x_scales;
  const void* values;       // or few rows' values [A, K], of the outputs' type
  const int32_t* offsets;   // [E + 1], or null: all rows are one expert's
  const int8_t *w, *w2;     // blocks of [E, K, N]; w2: the value weights
  const float *w_scales, *w2_scales;  // [E, N]
  int32_t E;
  int64_t A, K, N;
  void* out;          // [A, N]; hidden, act
  float *out2, *out3;  // gate, value; gelu' (null: not written)
  int32_t ntn;
};

struct Int8Tile {
  int32_t rows, cols;  // 0: no tiles, the weights are streamed
};
// int8_grad.hip: the tile of a gradient's product, K output columns.
Int8Tile int8_gradient_tile(int64_t E, int64_t A, int64_t K, int64_t cus);

// int8_few.hip: the product of few rows for each expert; and that of a few rows from
// their values (false where it does not take them).
void launch_int8_stream(const Int8Gemm& a, int epi, int dtype, hipStream_t s);
bool launch_int8_own(const Int8Gemm& a, int epi, int dtype, hipStream_t s);

namespace {

// Rows of expert e, clamped to [0, A] and non-decreasing whatever offsets holds.
__device__ __forceinline__ void int8_expert_rows(const Int8Gemm& a, int e, int64_t& r0,
                                                 int64_t& r1) {
  r0 = 0;
  r1 = a.A;
  if (a.offsets != nullptr) {
    const int64_t lo = a.offsets[e], hi = a.offsets[e + 1];
    r0 = lo < 0 ? 0 : lo > a.A ? a.A : lo;
    r1 = hi < r0 ? r0 : hi > a.A ? a.A : hi;
  }
}

// s_pref[e] = tiles of `rows` rows of the experts before e; ends with a barrier.
__device__ __forceinline__ void int8_row_tiles(const Int8Gemm& a, int rows, int32_t* s_pref) {
  if (threadIdx.x < kWave) {
    int carry = 0;
    for (int s = 0; s < a.E; s += kWave) {
      const int e = s + lane_id();
      int v = 0;
      if (e < a.E) {
        int64_t r0, r1;
        int8_expert_rows(a, e, r0, r1);
        v = (int)ceil_div(r1 - r0, rows);
      }
      const int incl = wave_incl_scan(v);
      if (e < a.E) s_pref[e + 1] = carry + incl;
      carry += __shfl(incl, kWave - 1, kWave);
    }
    if (lane_id() == 0) s_pref[0] = 0;
  }
  __syncthreads();
}

// e^-x and 1 / (1 + e^-x): for 16-bit results by the hardware's exponential and
// reciprocal (1 ulp each), for float32 ones by the library's.
template <typename T>
__device__ __forceinline__ float sigmoid_of(float x) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-x));
}
template <>
__device__ __forceinline__ float sigmoid_of<float>(float x) {
  return 1.f / (1.f + expf(-x));
}

// Phi(x) and exp(-x^2 / 2), relatively exact in both tails: 16-bit results by the
// fit of erfc, float32 ones by the library's erfc (1 + erf would cancel below 0).
template <typename T>
__device__ __forceinline__ float normal_cdf(float x, float& bell) {
  return norm_cdf(x, bell);
}
template <>
__device__ __forceinline__ float normal_cdf<float>(float x, float& bell) {
  bell = expf(-0.5f * x * x);
  return 0.5f * erfcf(x * -0.70710678118654752f);
}

// A product or sum that goes on to T, rounded to float32 first. Without the bar the compiler
// makes it and its rounding to float16 one operation in some columns of some kernels, and
// one value in thousands then depends on the kernel that the batch's size chose.
template <typename T>
__device__ __forceinline__ float in_float32(float v) {
  if constexpr (std::is_same<T, f16>::value) asm("" : "+v"(v));
  return v;
}
template <typename T>
__device__ __forceinline__ typename elem<T>::storage rounded(float v) {
  return to_bits<T>(in_float32<T>(v));
}

// The outputs of one column from its scaled sums p (and p2, the value). What a backward
// needs stays in float32: rounded to 16 bits it would be half of the gradient's error.
template <typename T, int EPI>
__device__ __forceinline__ void int8_epilogue(float p, float p2, typename elem<T>::storage& o,
                                              float& o2, float& o3) {
  if constexpr (EPI == kInt8Plain) {
    o = rounded<T>(p);
  } else if constexpr (EPI == kInt8SwiGLU) {
    o = rounded<T>(p * sigmoid_of<T>(p) * p2);
    o2 = p;
    o3 = p2;
  } else {
    float bell;
    const float c = normal_cdf<T>(p, bell);
    o = rounded<T>(p * c);
    o2 = fmaf(p, bell * 0.39894228040143268f, c);
  }
}

// n (at most 16) neighbouring columns of an output.
template <typename S>
__device__ __forceinline__ void int8_put(S* p, int n, const S (&o)[16]) {
  if (n == 16) {
    typedef S V __attribute__((ext_vector_type(16 / sizeof(S)), aligned(sizeof(S))));
    V v[sizeof(S)];
    __builtin_memcpy(v, o, sizeof(v));
#pragma unroll
    for (int j = 0; j < (int)sizeof(S); ++j)
      reinterpret_cast<V*>(p)[j] = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < n) p[j] = o[j];
  }
}

// n (at most 16) neighbouring values, zeros behind them.
__device__ __forceinline__ void int8_get(const float* p, int n, float (&v)[16]) {
  typedef float V __attribute__((ext_vector_type(16), aligned(4)));
  if (n == 16) {
    const V u = *reinterpret_cast<const V*>(p);
    __builtin_memcpy(v, &u, sizeof(v));
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = j < n ? p[j] : 0.f;
  }
}

}  // namespace
}  // namespace nt
