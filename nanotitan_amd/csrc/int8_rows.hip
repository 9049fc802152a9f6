// Rows and weights to 8-bit integers and back.
//
// Rows: a wave (or, where there are few rows or wide ones, a workgroup of four)
// holds a row in registers between finding its largest magnitude and rounding it,
// so it is read once. HBM bounds all of it.
//
// Weights: the channels' maxima run down the columns, so a pass over W finds them
// (an atomic max of magnitudes' bits: the order does not count) and a second one
// rounds. That one reads 64x64 blocks; a thread turns 4x4 values into four words
// of four reduction rows each, and the block's bytes turn in LDS.
#include <algorithm>

#include "int8.hpp"

namespace nt {
namespace {

constexpr int kVec = 16;  // columns of a lane at a time: 16 bytes of integers

template <typename T>
struct Sixteen {
  typedef typename elem<T>::storage S;
  typedef S V __attribute__((ext_vector_type(kVec), aligned(sizeof(S))));
  V v;
  // Columns c .. c + 15 of a row of f, zeros past its end.
  __device__ __forceinline__ void load(const S* row, int64_t c, int64_t f) {
    if (c + kVec <= f) {
      v = *reinterpret_cast<const V*>(row + c);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = c + i < f ? row[c + i] : S(0);
    }
  }
  __device__ __forceinline__ void store(S* row, int64_t c, int64_t f) const {
    if (c + kVec <= f) {
      *reinterpret_cast<V*>(row + c) = v;
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (c + i < f) row[c + i] = v[i];
    }
  }
  __device__ __forceinline__ uint32_t most() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const uint32_t b = abs_bits(elem<T>::load(v[i]));
      m = b > m ? b : m;
    }
    return m;
  }
  __device__ __forceinline__ uint4 codes(float s, float inv) const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = int8_code(elem<T>::load(v[4 * i + j]), s, inv);
      w[i] = pack_bytes(q[0], q[1], q[2], q[3]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ uint32_t wave_most(uint32_t m) {
#pragma unroll
  for (int o = kWave / 2; o >= 1; o >>= 1) {
    const uint32_t other = __shfl_xor(m, o, kWave);
    m = other > m ? other : m;
  }
  return m;
}

constexpr int kThreads = 256;

// TEAM lanes a row (64 or 256), C chunks of 16 columns a lane in registers; HELD
// false: rows past TEAM * C * 16 columns, read twice.
template <typename T, int TEAM, int C, bool HELD>
__global__ void __launch_bounds__(kThreads) int8_rows_kernel(const void* x, int64_t rows, int64_t f,
                                                             int8_t* codes, float* scales) {
  typedef typename elem<T>::storage S;
  __shared__ uint32_t s_most[kThreads / kWave];
  // (the grid has a second dimension: one holds 2^32 threads at most)
  const int64_t row =
      ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (kThreads / TEAM) + threadIdx.x / TEAM;
  const int lane = threadIdx.x % TEAM;
  if (row >= rows) return;  // with a workgroup a row: all its threads
  const int64_t pitch = int8_pitch(f);
  const S* in = static_cast<const S*>(x) + row * f;
  int8_t* out = codes + row * pitch;
  Sixteen<T> v[C];
  uint32_t m = 0;
  for (int64_t c0 = 0; c0 < (HELD ? 1 : pitch); c0 += TEAM * C * kVec) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i].load(in, c0 + (i * TEAM + lane) * kVec, f);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t b = v[i].most();
      m = b > m ? b : m;
    }
  }
  m = wave_most(m);
  if constexpr (TEAM > kWave) {
    if (lane_id() == 0) s_most[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TEAM / kWave; ++i) m = s_most[i] > m ? s_most[i] : m;
  }
  const float s = int8_scale(m), inv = int8_inverse(s);
  if (lane == 0) scales[row] = s;
  for (int64_t c0 = 0; c0 < (HELD ? 1 : pitch); c0 += TEAM * C * kVec) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int64_t c = c0 + (i * TEAM + lane) * kVec;
      if constexpr (!HELD) v[i].load(in, c, f);
      if (c < pitch) *reinterpret_cast<uint4*>(out + c) = v[i].codes(s, inv);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) int8_rows_decode_kernel(const int8_t* codes,
                                                                    const float* scales,
                                                                    int64_t rows, int64_t f,
                                                                    void* x) {
  typedef typename elem<T>::storage S;
  const int64_t chunks = ceil_div(f, (int64_t)kVec), pitch = int8_pitch(f);
  const int64_t total = rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / chunks, c = (i - row * chunks) * kVec;
    int8_t q[kVec];
    const uint4 w = *reinterpret_cast<const uint4*>(codes + row * pitch + c);
    __builtin_memcpy(q, &w, sizeof(q));
    const float s = scales[row];
    Sixteen<T> v;
#pragma unroll
    for (int j = 0; j < kVec; ++j) v.v[j] = int8_value<T>(q[j], s);
    v.store(static_cast<S*>(x) + row * f, c, f);
  }
}

// ------------------------------------------------------------------ weights

__global__ void __launch_bounds__(kThreads) int8_zero_kernel(uint32_t* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i < n) p[i] = 0;
}

// Maxima of 256 columns over `span` reduction rows: a thread has four columns, its
// wave 64 rows apart. Grid: column blocks, row spans, experts.
constexpr int kMostCols = 256;
template <typename T>
__global__ void __launch_bounds__(kThreads) int8_most_kernel(const void* W, int64_t K, int64_t N,
                                                             int64_t span, uint32_t* most) {
  typedef typename elem<T>::storage S;
  typedef S V4 __attribute__((ext_vector_type(4), aligned(sizeof(S))));
  const int64_t e = blockIdx.z, n = (int64_t)blockIdx.x * kMostCols + lane_id() * 4;
  const int64_t k0 = (int64_t)blockIdx.y * span, k1 = k0 + span < K ? k0 + span : K;
  if (n >= N) return;
  const S* w = static_cast<const S*>(W) + e * K * N + n;
  uint32_t m[4] = {0, 0, 0, 0};
  auto take = [&](int j, S v) {
    const uint32_t b = abs_bits(elem<T>::load(v));
    m[j] = b > m[j] ? b : m[j];
  };
  if (n + 4 <= N) {
#pragma unroll 8
    for (int64_t k = k0 + threadIdx.x / kWave; k < k1; k += kThreads / kWave) {
      const V4 v = *reinterpret_cast<const V4*>(w + k * N);
#pragma unroll
      for (int j = 0; j < 4; ++j) take(j, v[j]);
    }
  } else {
    for (int64_t k = k0 + threadIdx.x / kWave; k < k1; k += kThreads / kWave)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < N) take(j, w[k * N + j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n + j < N) atomicMax(&most[e * N + n + j], m[j]);
}

// Bytes of a block in LDS: [64 columns][64 reduction rows], a column's 64 bytes
// padded to 80, so that 16-byte reads stay aligned and columns spread over banks.
constexpr int kTurnPitch = 80;

// A 64x64 block to integers. Grid: column groups, reduction blocks, experts.
template <typename T>
__global__ void __launch_bounds__(kThreads) int8_weight_kernel(const void* W, int64_t K, int64_t N,
                                                               const uint32_t* most, int8_t* codes,
                                                               float* scales) {
  typedef typename elem<T>::storage S;
  typedef S V4 __attribute__((ext_vector_type(4), aligned(sizeof(S))));
  __shared__ __attribute__((aligned(16))) int8_t s_turn[kInt8Block * kTurnPitch];
  const int64_t e = blockIdx.z, n0 = (int64_t)blockIdx.x * kInt8Block;
  const int64_t k0 = (int64_t)blockIdx.y * kInt8Block;
  const int c = threadIdx.x % 16 * 4, r = threadIdx.x / 16 * 4;
  const S* w = static_cast<const S*>(W) + e * K * N + n0 + c;
  float s[4], inv[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s[j] = int8_scale(n0 + c + j < N ? most[e * N + n0 + c + j] : 0u);
    inv[j] = int8_inverse(s[j]);
    if (blockIdx.y == 0 && r == 0 && n0 + c + j < N) scales[e * N + n0 + c + j] = s[j];
  }
  int q[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    V4 v;
    const int64_t k = k0 + r + i;
    if (k < K && n0 + c + 4 <= N) {
      v = *reinterpret_cast<const V4*>(w + k * N);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = k < K && n0 + c + j < N ? w[k * N + j] : S(0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) q[i][j] = int8_code(elem<T>::load(v[j]), s[j], inv[j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint32_t*>(s_turn + (c + j) * kTurnPitch + r) =
        pack_bytes(q[0][j], q[1][j], q[2][j], q[3][j]);
  __syncthreads();
  // thread: operand t, lane (g, i)
  const int t = threadIdx.x / kWave, g = threadIdx.x % kWave / 16, i = threadIdx.x % 16;
  const int col = 16 * (i / 4) + 4 * t + i % 4;
  const int64_t block = (e * int8_groups(N) + blockIdx.x) * (int8_pitch(K) / kInt8Block) +
                        blockIdx.y;
  *reinterpret_cast<uint4*>(codes + block * kInt8Block * kInt8Block + threadIdx.x * 16) =
      *reinterpret_cast<const uint4*>(s_turn + col * kTurnPitch + g * 16);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) int8_weight_decode_kernel(const int8_t* codes,
                                                                      const float* scales,
                                                                      int64_t K, int64_t N,
                                                                      void* W) {
  typedef typename elem<T>::storage S;
  typedef S V4 __attribute__((ext_vector_type(4), aligned(sizeof(S))));
  __shared__ __attribute__((aligned(16))) int8_t s_turn[kInt8Block * kTurnPitch];
  const int64_t e = blockIdx.z, n0 = (int64_t)blockIdx.x * kInt8Block;
  const int64_t k0 = (int64_t)blockIdx.y * kInt8Block;
  const int t = threadIdx.x / kWave, g = threadIdx.x % kWave / 16, i = threadIdx.x % 16;
  const int col = 16 * (i / 4) + 4 * t + i % 4;
  const int64_t block = (e * int8_groups(N) + blockIdx.x) * (int8_pitch(K) / kInt8Block) +
                        blockIdx.y;
  *reinterpret_cast<uint4*>(s_turn + col * kTurnPitch + g * 16) =
      *reinterpret_cast<const uint4*>(codes + block * kInt8Block * kInt8Block + threadIdx.x * 16);
  __syncthreads();
  const int c = threadIdx.x % 16 * 4, r = threadIdx.x / 16 * 4;
  S* w = static_cast<S*>(W) + e * K * N + n0 + c;
  V4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float s = n0 + c + j < N ? scales[e * N + n0 + c + j] : 0.f;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(s_turn + (c + j) * kTurnPitch + r);
#pragma unroll
    for (int b = 0; b < 4; ++b) v[b][j] = int8_value<T>((int8_t)(word >> (8 * b)), s);
  }
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int64_t k = k0 + r + b;
    if (k >= K) break;
    if (n0 + c + 4 <= N) {
      *reinterpret_cast<V4*>(w + k * N) = v[b];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + c + j < N) w[k * N + j] = v[b][j];
    }
  }
}

int check_rows(int dtype, int64_t rows, int64_t f) {
  if (!int8_float(dtype)) return NT_ERR_DTYPE;
  if (rows < 0 || f < 1) return NT_ERR_INVALID_ARG;
  if (rows > INT32_MAX || f > kInt8MaxK) return NT_ERR_TOO_LARGE;
  return NT_OK;
}
int check_weight(int dtype, int32_t E, int64_t K, int64_t N) {
  if (!int8_float(dtype)) return NT_ERR_DTYPE;
  if (E < 1 || K < 1 || N < 1) return NT_ERR_INVALID_ARG;
  if (E > NT_MAX_EXPERTS) return NT_ERR_TOO_MANY_EXPERTS;
  if (K > kInt8MaxK || N > 1 << 22) return NT_ERR_TOO_LARGE;
  return NT_OK;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int64_t nt_int8_pitch(int64_t f) { return f < 0 ? 0 : int8_pitch(f); }

size_t nt_int8_weight_bytes(int32_t E, int64_t K, int64_t N) {
  if (check_weight(NT_F32, E, K, N) != NT_OK) return 0;
  return (size_t)E * int8_matrix(K, N);
}

int nt_int8_rows(int dtype, const void* x, int64_t rows, int64_t f, int8_t* codes, float* scales,
                 hipStream_t stream) {
  const int st = check_rows(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  if (x == nullptr || codes == nullptr || scales == nullptr || !aligned16(codes))
    return NT_ERR_INVALID_ARG;
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    auto launch = [&](auto kernel, int team) {
      const int64_t blocks = ceil_div(rows, (int64_t)(kThreads / team)), wide = 1 << 23;
      hipLaunchKernelGGL(kernel,
                         dim3((unsigned)std::min(blocks, wide), (unsigned)ceil_div(blocks, wide)),
                         dim3(kThreads), 0, stream, x, rows, f, codes, scales);
    };
    const int64_t chunks = ceil_div(f, (int64_t)kVec);
    if (chunks <= 64) launch(int8_rows_kernel<T, 64, 1, true>, 64);
    else if (chunks <= 128 && rows >= 1024) launch(int8_rows_kernel<T, 64, 2, true>, 64);
    else if (chunks <= 256) launch(int8_rows_kernel<T, 256, 1, true>, 256);
    else if (chunks <= 512) launch(int8_rows_kernel<T, 256, 2, true>, 256);
    else if (chunks <= 1024) launch(int8_rows_kernel<T, 256, 4, true>, 256);
    else launch(int8_rows_kernel<T, 256, 4, false>, 256);
  });
  return launch_status();
}

int nt_int8_rows_decode(int dtype, const int8_t* codes, const float* scales, int64_t rows,
                        int64_t f, void* x, hipStream_t stream) {
  const int st = check_rows(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  if (x == nullptr || codes == nullptr || scales == nullptr || !aligned16(codes))
    return NT_ERR_INVALID_ARG;
  const int64_t blocks = ceil_div(rows * ceil_div(f, (int64_t)kVec), (int64_t)kThreads);
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    hipLaunchKernelGGL((int8_rows_decode_kernel<T>),
                       dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(kThreads), 0,
                       stream, codes, scales, rows, f, x);
  });
  return launch_status();
}

size_t nt_int8_weight_workspace_bytes(int32_t E, int64_t N) {
  return check_weight(NT_F32, E, 1, N) == NT_OK ? (size_t)E * N * 4 : 0;
}

int nt_int8_weight(int dtype, const void* W, int32_t E, int64_t K, int64_t N, int8_t* codes,
                   float* scales, void* ws, size_t ws_bytes, hipStream_t stream) {
  const int st = check_weight(dtype, E, K, N);
  if (st != NT_OK) return st;
  if (W == nullptr || codes == nullptr || scales == nullptr || !aligned16(codes))
    return NT_ERR_INVALID_ARG;
  if (ws == nullptr || ws_bytes < nt_int8_weight_workspace_bytes(E, N) ||
      reinterpret_cast<uintptr_t>(ws) % 4 != 0)
    return NT_ERR_WORKSPACE;
  uint32_t* most = static_cast<uint32_t*>(ws);
  hipLaunchKernelGGL(int8_zero_kernel, dim3((unsigned)ceil_div((int64_t)E * N, (int64_t)kThreads)),
                     dim3(kThreads), 0, stream, most, (int64_t)E * N);
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    const int64_t span = 256;
    hipLaunchKernelGGL((int8_most_kernel<T>),
                       dim3((unsigned)ceil_div(N, (int64_t)kMostCols),
                            (unsigned)ceil_div(K, span), (unsigned)E),
                       dim3(kThreads), 0, stream, W, K, N, span, most);
    hipLaunchKernelGGL((int8_weight_kernel<T>),
                       dim3((unsigned)int8_groups(N), (unsigned)(int8_pitch(K) / kInt8Block),
                            (unsigned)E),
                       dim3(kThreads), 0, stream, W, K, N, most, codes, scales);
  });
  return launch_status();
}

int nt_int8_weight_decode(int dtype, const int8_t* codes, const float* scales, int32_t E,
                          int64_t K, int64_t N, void* W, hipStream_t stream) {
  const int st = check_weight(dtype, E, K, N);
  if (st != NT_OK) return st;
  if (W == nullptr || codes == nullptr || scales == nullptr || !aligned16(codes))
    return NT_ERR_INVALID_ARG;
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    hipLaunchKernelGGL((int8_weight_decode_kernel<T>),
                       dim3((unsigned)int8_groups(N),
                            (unsigned)ceil_div(K, (int64_t)kInt8Block), (unsigned)E),
                       dim3(kThreads), 0, stream, codes, scales, K, N, W);
  });
  return launch_status();
}

}  // extern "C"
