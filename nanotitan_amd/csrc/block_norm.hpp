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
// The raw values with those that the chunk does not own cleared: 16-bit ones by
// pairs.
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> owned(const Raw<T, V>& raw, const Chunk<V>& c) {
  Raw<T, V> out = raw;
  if constexpr (sizeof(raw[0]) == 2 && V % 2 == 0) {
    typedef uint32_t Pairs __attribute__((ext_vector_type(V / 2)));
    Pairs p = __builtin_bit_cast(Pairs, raw);
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      p[i] &= (c.owns(2 * i) ? 0xffffu : 0u) | (c.owns(2 * i + 1) ? 0xffff0000u : 0u);
    out = __builtin_bit_cast(Raw<T, V>, p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = c.owns(i) ? raw[i] : 0;
  }
  return out;
}
// The values as they are, and zero where the chunk does not own them.
template <typename T, int V>
__device__ __forceinline__ void all_values(const Raw<T, V>& raw, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = elem<T>::load(raw[i]);
}
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

// v plus another lane's, by its place in a row of 16 lanes.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float plus_lane(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf,
                                                        ROWS == 0xf));
}
// Sum over each LANES neighbouring lanes, which all receive it.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(LANES <= 16, "a row of lanes");
  if constexpr (LANES >= 2) v = plus_lane<0xb1>(v);   // lane ^ 1
  if constexpr (LANES >= 4) v = plus_lane<0x4e>(v);   // lane ^ 2
  if constexpr (LANES >= 8) v = plus_lane<0x141>(v);  // 7 - lane, of each 8
  if constexpr (LANES >= 16) v = plus_lane<0x140>(v); // 15 - lane, of each 16
  return v;
}
// Sum over the wave: in its last lane.
__device__ __forceinline__ float last_lane_sum(float v) {
  v = lanes_sum<16>(v);
  v = plus_lane<0x142, 0xa>(v);  // lane 15 of a row to the next, rows 1 and 3
  return plus_lane<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
}

// Sums over the TPR threads of a row, every thread receiving them: inside a
// wave by lane moves (shuffles through LDS took a fifth of a row's
// instructions), then through LDS across the row's waves, which have the
// workgroup alone. Calls alternate between the halves of s_red ([2][kMost]
// [waves]), so that one barrier each is enough.
template <int TPR, int MOST>
struct RowSum {
  static constexpr int W = TPR > kWave ? TPR / kWave : 1;
  static constexpr int kSize = 2 * MOST * W;
  float* s_red;
  int half = 0;
  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N]) {
    static_assert(N <= MOST && (TPR == 16 || TPR >= kWave), "row sums");
    if constexpr (TPR == 16) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = lanes_sum<16>(v[i]);
    } else if constexpr (TPR == kWave) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(last_lane_sum(v[i])), 63));
    } else {
      float* s = s_red + half * MOST * W;
      half ^= 1;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = last_lane_sum(v[i]);
      if (lane_id() == kWave - 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i * W + threadIdx.x / kWave] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = lanes_sum<W>(s[i * W + lane_id() % W]);
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
