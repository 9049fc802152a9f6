// Values in 8-bit integers: the scale, the rounding and the layouts that the
// int8 kernels share.
//
// A row of activations (or an output channel of weights) v is held as s q with
//   s = max(max|v| / 127, 2^-126) in float32,  q = the integer nearest to v / s,
// ties to even, so |q| <= 127. The division is exact in its decision (int8_code),
// not a product with a rounded reciprocal: half-way values are common in 16-bit
// rows (half the row's largest value is one), and which way they go would
// otherwise depend on the code that computes them. A row that holds an infinity or
// a NaN has a NaN scale and integers 0: all that is computed from it is NaN.
#pragma once

#include "common.hpp"
#include "nanotitan_int8.h"

namespace nt {

constexpr int kInt8Block = 64;   // columns and reduction rows of a weight block
constexpr int kInt8Pitch = 128;  // reduction rows are padded with zeros to this: the widest k-step
// 127 * 127 * kInt8MaxK < 2^31: an int32 sum cannot overflow
constexpr int64_t kInt8MaxK = NT_INT8_MAX_K;
constexpr int64_t kInt8MaxRows = NT_INT8_MAX_ROWS;  // 256 threads each are a launch's 2^32

// Integers lie in operands of a 16x16x64 matrix instruction, 1 KiB each: [g][i][16]
// holds, lane 16 g + i by lane, values 16 g .. 16 g + 15 of a step's 64 of row (or
// column) i. A wave's 16-byte loads then read 1 KiB on end, from memory or from LDS
// (where that is free of bank conflicts), whichever 64 values of a row it takes.
// Activations [A, K]: 16 rows after another,
//   codes[a / 16][k / 64][g][a % 16][k % 16],  g = k % 64 / 16.
// Weights [E, K, N]: the four operands of 64 columns together,
//   codes[e][n / 64][k / 64][t][g][i][k % 16],  n % 64 = 16 (i / 4) + 4 t + i % 4.
// Which 16 of the 64 columns make operand t is chosen for the result: lane 16 g +
// r of the instruction holds 4 values of row r, and over the four t they are 16
// neighbouring columns. K is padded with zeros to a multiple of 128 (the longest
// k-step), N to one of 64; activations' rows past the last, up to 16, hold anything.
__host__ __device__ constexpr int64_t int8_pitch(int64_t k) { return round_up(k, kInt8Pitch); }
// Bytes of A rows, and where row a begins (its 16-byte pieces are 256 bytes apart).
__host__ __device__ constexpr int64_t int8_rows_bytes(int64_t A, int64_t pitch) {
  return round_up(A, 16) * pitch;
}
__host__ __device__ constexpr int64_t int8_row(int64_t a, int64_t pitch) {
  return (a >> 4) * 16 * pitch + (a & 15) * 16;
}
__host__ __device__ constexpr int64_t int8_groups(int64_t n) { return ceil_div(n, kInt8Block); }
__host__ __device__ constexpr int64_t int8_matrix(int64_t K, int64_t N) {
  return int8_groups(N) * kInt8Block * int8_pitch(K);
}

// The scale of values whose largest magnitude has these bits.
__device__ __forceinline__ float int8_scale(uint32_t most) {
  if (most >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const float s = __fdiv_rn(__uint_as_float(most), 127.f);
  return s < 0x1p-126f ? 0x1p-126f : s;
}
// 1 / s for int8_code; 0 for a NaN scale, which makes every integer 0.
__device__ __forceinline__ float int8_inverse(float s) { return s == s ? 1.f / s : 0.f; }

// The integer nearest to x / s, ties to even, for |x| <= 127.5 s. x * inv is off
// by less than 2^-15, so the first guess is the nearest integer or, next to a
// border, its neighbour. x - r s is exact where it decides: r s has at most 31
// bits, and the difference is below 1.01 s and a multiple of both operands'
// last bits.
__device__ __forceinline__ int int8_code(float x, float s, float inv) {
  const float r = rintf(x * inv);
  const float off = fmaf(-r, s, x), half = 0.5f * s;
  int q = (int)r;
  if (fabsf(off) >= half) {
    const bool odd = q & 1;
    if (off > half || (off == half && odd)) q += 1;
    else if (off < -half || (off == -half && odd)) q -= 1;
  }
  return inv == 0.f ? 0 : q;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t pack_bytes(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 |
         (uint32_t)d << 24;
}

// q s in T: rounded once; a value that rounds past the type's largest is that.
template <typename T>
struct int8_most;
template <>
struct int8_most<float> {
  static constexpr float value = 0x1.fffffep127f;
};
template <>
struct int8_most<bf16> {
  static constexpr float value = 0x1.fep127f;
};
template <>
struct int8_most<f16> {
  static constexpr float value = 65504.f;
};
template <typename T>
__device__ __forceinline__ typename elem<T>::storage int8_value(int q, float s) {
  const float v = (float)q * s, most = int8_most<T>::value;
  return elem<T>::store(v > most ? most : v < -most ? -most : v);  // (a NaN stays one)
}

constexpr int kVec = 16;  // values of a 16-byte piece of integers

// N (8 or 16) neighbouring values of a row.
template <typename T, int N = kVec>
struct Some {
  typedef typename elem<T>::storage S;
  typedef S V __attribute__((ext_vector_type(N), aligned(sizeof(S))));
  V v;
  // Columns c .. c + N - 1 of a row of f, zeros past its end.
  __device__ __forceinline__ void load(const S* row, int64_t c, int64_t f) {
    if (c + N <= f) {
      v = *reinterpret_cast<const V*>(row + c);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = c + i < f ? row[c + i] : S(0);
    }
  }
  __device__ __forceinline__ void store(S* row, int64_t c, int64_t f) const {
    if (c + N <= f) {
      *reinterpret_cast<V*>(row + c) = v;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < f) row[c + i] = v[i];
    }
  }
  __device__ __forceinline__ uint32_t most() const {
    if constexpr (sizeof(S) == 2) {
      // pairs at once: magnitudes' bits order as the values do
      typedef unsigned short U2 __attribute__((ext_vector_type(2)));
      uint32_t w[N / 2];
      __builtin_memcpy(w, &v, sizeof(w));
      U2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(U2, w[i] & 0x7fff7fffu));
      return abs_bits(elem<T>::load(m[0] > m[1] ? m[0] : m[1]));
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t b = abs_bits(elem<T>::load(v[i]));
        m = b > m ? b : m;
      }
      return m;
    }
  }
  // x / s by the inverse, plus 1.5 2^23: the sum's low byte is the nearest integer,
  // or next to a border its neighbour, which x minus s times it tells. Then
  // int8_code decides; of normal values in bf16 one group of 1,024 in thirty.
  typedef uint32_t Codes __attribute__((ext_vector_type(N / 4)));
  __device__ __forceinline__ Codes codes(float s, float inv) const {
    constexpr float kMagic = 12582912.f;
    Codes w;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      uint32_t t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = elem<T>::load(v[4 * i + j]), sum = fmaf(x, inv, kMagic);
        most = fmaxf(most, fabsf(fmaf(kMagic - sum, s, x)));
        t[j] = __float_as_uint(sum);
      }
      w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[3], t[2], 0x0c0c0400u),
                                   __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u), 0x05040100u);
    }
    if (!(most < 0.5f * s) || inv == 0.f) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        int q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = int8_code(elem<T>::load(v[4 * i + j]), s, inv);
        w[i] = pack_bytes(q[0], q[1], q[2], q[3]);
      }
    }
    return w;
  }
};

inline bool int8_float(int dtype) { return dtype == NT_F32 || dtype == NT_F16 || dtype == NT_BF16; }

// f(type tag) for an activation type.
template <typename T>
struct tag {
  typedef T type;
};
template <typename F>
inline void int8_by_type(int dtype, F&& f) {
  if (dtype == NT_F32) f(tag<float>());
  else if (dtype == NT_F16) f(tag<f16>());
  else f(tag<bf16>());
}

}  // namespace nt
