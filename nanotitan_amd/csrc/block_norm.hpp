// What the block norms' forward and backward share: how a row lies in the
// threads, its loads and sums, and the choice of kernel by width and type.
#pragma once

#include <algorithm>
#include <type_traits>

#include "bits.hpp"
#include "common.hpp"

namespace nt {
namespace norm {

// A row's threads hold CH chunks of V columns each, the chunks interleaved over
// the threads. Rows of up to a wave's threads share a workgroup with others, a
// wider one has it alone.
constexpr int kVec = 8;
constexpr int kMaxThreads = 1024;
constexpr int64_t kMaxWidth = 2 * kMaxThreads * kVec;
constexpr int block_threads(int row_threads) { return row_threads <= kWave ? 256 : row_threads; }

// Columns start .. start + V - 1 of a row of d, of which the first `skip` are
// another chunk's: a chunk that would reach past the end starts earlier
// instead, so that every load is whole and needs no branch.
template <int V>
struct Chunk {
  int32_t start, skip;
  Chunk() = default;
  __device__ __forceinline__ Chunk(int32_t c0, int32_t d) {
    start = c0 + V <= d ? c0 : d - V;
    skip = c0 - start;
  }
  __device__ __forceinline__ bool owns(int i) const { return i >= skip; }
};

template <typename T, int V>
using Raw = typename elem<T>::storage __attribute__((ext_vector_type(V),
                                                     aligned(sizeof(typename elem<T>::storage))));

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const void* rows, int64_t base, const Chunk<V>& c) {
  return *reinterpret_cast<const Raw<T, V>*>(
      static_cast<const typename elem<T>::storage*>(rows) + base + c.start);
}
// The values, zero where the chunk does not own them.
template <typename T, int V>
__device__ __forceinline__ void values(const Raw<T, V>& raw, const Chunk<V>& c, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = c.owns(i) ? elem<T>::load(raw[i]) : 0.f;
}
template <typename T, int V>
__device__ __forceinline__ void store_chunk(void* rows, int64_t base, const Chunk<V>& c,
                                            const float (&v)[V]) {
  typename elem<T>::storage* p = static_cast<typename elem<T>::storage*>(rows) + base + c.start;
  Raw<T, V> raw;
#pragma unroll
  for (int i = 0; i < V; ++i) raw[i] = to_bits<T>(v[i]);
  if (c.skip == 0) {
    *reinterpret_cast<Raw<T, V>*>(p) = raw;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c.owns(i)) p[i] = raw[i];
  }
}

// Parameters come in one type of their own, read once per thread; `none` where
// there are none, zero where the chunk does not own a column.
__device__ __forceinline__ float load_param(const void* p, int dt, int64_t i) {
  if (dt == NT_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return dt == NT_BF16 ? bf16_to_f32(v) : f16_to_f32(v);
}
__device__ __forceinline__ void store_param(void* p, int dt, int64_t i, float v) {
  if (dt == NT_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = dt == NT_BF16 ? f32_to_bf16(v) : f32_to_f16(v);
}
template <int V>
__device__ __forceinline__ void load_params(const void* p, int dt, const Chunk<V>& c, float none,
                                            float (&v)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = c.owns(i) ? none : 0.f;
  } else if (dt == NT_F32) {
    values<float, V>(load_raw<float, V>(p, 0, c), c, v);
  } else if (dt == NT_BF16) {
    values<bf16, V>(load_raw<bf16, V>(p, 0, c), c, v);
  } else {
    values<f16, V>(load_raw<f16, V>(p, 0, c), c, v);
  }
}

// s w and s b, all that a row needs of the scale (one value or one a column),
// the weight and the bias: p = s (vhat w + b) = vhat (s w) + s b.
template <int V, bool LAYER>
__device__ __forceinline__ void load_scaled(const void* w, const void* b, const void* scale,
                                            int32_t scale_cols, int dt, const Chunk<V>& c,
                                            float (&sw)[V], float (&sb)[V]) {
  const float one = scale != nullptr && scale_cols == 1 ? load_param(scale, dt, 0) : 1.f;
  float s[V];
  load_params<V>(scale_cols == 1 ? nullptr : scale, dt, c, one, s);
  load_params<V>(w, dt, c, 1.f, sw);
  if constexpr (LAYER) load_params<V>(b, dt, c, 0.f, sb);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    sw[i] *= s[i];
    if constexpr (LAYER) sb[i] *= s[i];
  }
}

// Sums over the TPR threads of a row, every thread receiving them: shuffles
// inside a wave, then LDS across the row's waves (which have the workgroup
// alone). Calls alternate between the halves of s_red ([2][N][waves]), so that
// one barrier each is enough.
template <int TPR, int N>
struct RowSum {
  float* s_red;
  int half = 0;
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int o = (TPR < kWave ? TPR : kWave) / 2; o >= 1; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o, kWave);
    if constexpr (TPR > kWave) {
      constexpr int W = TPR / kWave;
      float* s = s_red + half * N * W;
      half ^= 1;
      if (lane_id() == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i * W + threadIdx.x / kWave] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v[i] += s[i * W + w];
      }
    }
  }
};

// The layouts: V columns a chunk, TPR threads a row, CH chunks a thread.
template <int V_, int TPR_, int CH_>
struct Shape {
  static constexpr int V = V_, TPR = TPR_, CH = CH_;
};
// f(shape) for a width: the fewest threads that hold it eight columns each, in
// a coarse set (16, 64, then powers of two) to keep the kernels few.
template <typename F>
void by_width(int64_t d, F&& f) {
  if (d < kVec) f(Shape<1, 16, 1>());
  else if (d <= 16 * kVec) f(Shape<8, 16, 1>());
  else if (d <= 64 * kVec) f(Shape<8, 64, 1>());
  else if (d <= 128 * kVec) f(Shape<8, 128, 1>());
  else if (d <= 256 * kVec) f(Shape<8, 256, 1>());
  else if (d <= 512 * kVec) f(Shape<8, 512, 1>());
  else if (d <= 1024 * kVec) f(Shape<8, 1024, 1>());
  else f(Shape<8, 1024, 2>());
}

template <typename F>
int by_types(int x_dtype, int dtype, F&& f) {
  if (x_dtype == NT_F32 && dtype == NT_F32) return f(float(), float());
  if (x_dtype == NT_BF16 && dtype == NT_BF16) return f(bf16(), bf16());
  if (x_dtype == NT_F16 && dtype == NT_F16) return f(f16(), f16());
  if (x_dtype == NT_F32 && dtype == NT_BF16) return f(float(), bf16());
  if (x_dtype == NT_F32 && dtype == NT_F16) return f(float(), f16());
  return NT_ERR_DTYPE;
}

// What a row's work reads besides x or h: nothing, y, or y and a gate value
// for every element. (A kernel each: absent loads cost registers and waits.)
enum Mode { kPre = 0, kPost = 1, kGated = 2 };
template <typename F>
void by_mode(bool y, bool gate, F&& f) {
  if (!y) f(std::integral_constant<int, kPre>());
  else if (!gate) f(std::integral_constant<int, kPost>());
  else f(std::integral_constant<int, kGated>());
}

// Workgroups: all resident at once (`waves` a SIMD on 256 CUs), each with every
// so-manieth row. By the sizes alone: the order of the parameters' sums in the
// backward is the same on every device.
inline int64_t blocks_of(int64_t T, int64_t d, int waves) {
  int64_t n = 1;
  by_width(d, [&](auto s) {
    constexpr int TPR = decltype(s)::TPR;
    n = std::min<int64_t>(waves * 256 * 256 / block_threads(TPR),
                          ceil_div(T, (int64_t)(block_threads(TPR) / TPR)));
  });
  return std::max<int64_t>(1, n);
}

inline int check_norm(int x_dtype, int dtype, int param, int kind, int64_t T, int64_t d) {
  if (by_types(x_dtype, dtype, [](auto, auto) { return (int)NT_OK; }) != NT_OK) return NT_ERR_DTYPE;
  if (param != NT_F32 && param != NT_F16 && param != NT_BF16) return NT_ERR_DTYPE;
  if ((kind != NT_NORM_RMS && kind != NT_NORM_LAYER) || T < 0 || d < 1) return NT_ERR_INVALID_ARG;
  if (d > kMaxWidth || T > INT32_MAX) return NT_ERR_TOO_LARGE;
  return NT_OK;
}

}  // namespace norm
}  // namespace nt
