// Rows and weights to 8-bit integers and back.
//
// Rows: a team of lanes holds a row in registers between finding its largest
// magnitude and rounding it, so it is read once. A workgroup takes eight rows (four
// wide ones), whose integers pass through LDS: in memory the 16-byte pieces of 16
// rows alternate, and eight of them make a 128-byte line (written piece by piece,
// 32,768 rows of 14,336 took 534 us for 235 in row order). Rounding one value has to
// stay near seven instructions for HBM to bound the kernel (Some::codes). Few
// rows take a workgroup each and write their pieces as they are.
//
// Weights: the channels' maxima run down the columns, so a pass over W finds them
// (an atomic max of magnitudes' bits: the order does not count) and a second one
// rounds. A thread turns 4x4 values into four words of four reduction rows each, and
// a block's bytes turn in LDS.
#include <algorithm>

#include "int8.hpp"

namespace nt {
namespace {

constexpr int kThreads = 256;

// ROWS rows a workgroup, TEAM lanes a row, C chunks of 8 columns a lane in
// registers (a wave's loads of 16-bit values are then 1 KiB on end); HELD false: rows
// past TEAM * C * 8 columns, read twice. Workgroups b
// and b + 8 share an XCD and so an L2: the parts of a block of 16 rows go to such.
template <typename T, int ROWS, int TEAM, int C, bool HELD>
__global__ void __launch_bounds__(ROWS* TEAM)
    int8_rows_kernel(const void* x, int64_t rows, int64_t f, int8_t* codes, float* scales) {
  typedef typename elem<T>::storage S;
  constexpr int G = C % 4 == 0 ? 4 : C % 2 == 0 ? 2 : 1;  // chunks of a lane that turn at once
  // the rows' pieces of 16 columns, padded so that neighbours begin in other banks
  constexpr int kPitch = ROWS * 16 + 16, kParts = 16 / ROWS, kPieces = G * TEAM / 2;
  __shared__ __attribute__((aligned(16))) char s_turn[2][kPieces * kPitch];
  const int64_t b = blockIdx.x;
  const int64_t row0 = (b / (8 * kParts) * 8 + b % 8) * 16 + b / 8 % kParts * ROWS;
  if (row0 >= rows) return;
  const int r = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
  const bool live = row0 + r < rows;
  const int64_t row = live ? row0 + r : rows - 1;  // past the last: that one again
  const int64_t pitch = int8_pitch(f);
  const int chunks = (int)(pitch / 8);
  const S* in = static_cast<const S*>(x) + row * f;
  typedef Some<T, 8> Chunk;
  Chunk v[C];
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (c0 + i * TEAM < chunks) v[i].load(in, (int64_t)(c0 + i * TEAM + lane) * 8, f);
  };
  uint32_t m = 0;
  for (int c0 = 0; c0 < (HELD ? 1 : chunks); c0 += TEAM * C) {
    load(c0);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t most = c0 + i * TEAM < chunks ? v[i].most() : 0u;
      m = most > m ? most : m;
    }
  }
#pragma unroll
  for (int o = (TEAM < kWave ? TEAM : kWave) / 2; o >= 1; o >>= 1) {
    const uint32_t other = __shfl_xor(m, o, kWave);
    m = other > m ? other : m;
  }
  if constexpr (TEAM > kWave) {
    __shared__ uint32_t s_most[ROWS * TEAM / kWave];
    if (lane_id() == 0) s_most[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TEAM / kWave; ++i) {
      const uint32_t other = s_most[r * (TEAM / kWave) + i];
      m = other > m ? other : m;
    }
  }
  const float s = int8_scale(m), inv = int8_inverse(s);
  if (lane == 0 && live) scales[row] = s;
  // thread: row threadIdx % ROWS of piece threadIdx / ROWS
  int8_t* out = codes + int8_row(row0 + threadIdx.x % ROWS, pitch);
  int buffer = 0;
  for (int c0 = 0; c0 < (HELD ? 1 : chunks); c0 += TEAM * C) {
    if constexpr (!HELD) load(c0);
#pragma unroll
    for (int i = 0; i < C; i += G) {
      if (c0 + i * TEAM >= chunks) break;
      char* turn = s_turn[buffer];
      buffer ^= 1;
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (c0 + (i + g) * TEAM < chunks)
          *reinterpret_cast<typename Chunk::Codes*>(turn + (g * TEAM + lane) / 2 * kPitch + r * 16 +
                                                    lane % 2 * 8) = v[i + g].codes(s, inv);
      __syncthreads();
#pragma unroll
      for (int at = threadIdx.x / ROWS; at < kPieces; at += TEAM) {
        const int c = (c0 + i * TEAM) / 2 + at;
        if (c < chunks / 2)
          *reinterpret_cast<uint4*>(out + (int64_t)c * 256) =
              *reinterpret_cast<const uint4*>(turn + at * kPitch + threadIdx.x % ROWS * 16);
      }
    }
  }
}

// A row a workgroup.
template <typename T, int C, bool HELD>
__global__ void __launch_bounds__(kThreads)
    int8_row_kernel(const void* x, int64_t f, int8_t* codes, float* scales) {
  typedef typename elem<T>::storage S;
  __shared__ uint32_t s_most[kThreads / kWave];
  const int64_t row = blockIdx.x, pitch = int8_pitch(f);
  const int lane = threadIdx.x;
  const S* in = static_cast<const S*>(x) + row * f;
  int8_t* out = codes + int8_row(row, pitch);
  Some<T> v[C];
  uint32_t m = 0;
  for (int64_t c0 = 0; c0 < (HELD ? 1 : pitch); c0 += kThreads * C * kVec) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i].load(in, c0 + (i * kThreads + lane) * kVec, f);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t most = v[i].most();
      m = most > m ? most : m;
    }
  }
#pragma unroll
  for (int o = kWave / 2; o >= 1; o >>= 1) {
    const uint32_t other = __shfl_xor(m, o, kWave);
    m = other > m ? other : m;
  }
  if (lane_id() == 0) s_most[threadIdx.x / kWave] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / kWave; ++i) m = s_most[i] > m ? s_most[i] : m;
  const float s = int8_scale(m), inv = int8_inverse(s);
  if (lane == 0) scales[row] = s;
  for (int64_t c0 = 0; c0 < (HELD ? 1 : pitch); c0 += kThreads * C * kVec) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int64_t c = c0 + (i * kThreads + lane) * kVec;
      if constexpr (!HELD) v[i].load(in, c, f);
      if (c < pitch)
        *reinterpret_cast<typename Some<T>::Codes*>(out + c * 16) = v[i].codes(s, inv);
    }
  }
}

// 16 rows by 64 chunks a workgroup, a lane a chunk of four rows: the rows' pieces lie
// in lines that its waves read one after the other, its writes are whole lines.
template <typename T>
__global__ void __launch_bounds__(kThreads) int8_rows_decode_kernel(const int8_t* codes,
                                                                    const float* scales,
                                                                    int64_t rows, int64_t f,
                                                                    void* x) {
  typedef typename elem<T>::storage S;
  const int64_t pitch = int8_pitch(f), c = ((int64_t)blockIdx.y * kWave + lane_id()) * kVec;
  if (c >= f) return;
  const int64_t row0 = (int64_t)blockIdx.x * 16 + threadIdx.x / kWave * 4;
  const int8_t* in = codes + int8_row(row0, pitch) + c * 16;
  uint4 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint4*>(in)[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (row0 + i >= rows) break;
    int8_t q[kVec];
    __builtin_memcpy(q, &w[i], sizeof(q));
    const float s = scales[row0 + i];
    Some<T> v;
#pragma unroll
    for (int j = 0; j < kVec; ++j) v.v[j] = int8_value<T>(q[j], s);
    v.store(static_cast<S*>(x) + (row0 + i) * f, c, f);
  }
}

// ------------------------------------------------------------------ weights

__global__ void __launch_bounds__(kThreads) int8_zero_kernel(uint32_t* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i < n) p[i] = 0;
}

// Maxima of `span` reduction rows: a lane has 16 bytes of columns (kMostBytes a
// wave), its workgroup's waves are rows apart. Grid: column blocks, row spans,
// experts.
constexpr int kMostBytes = kWave * 16;
template <typename T>
__global__ void __launch_bounds__(kThreads) int8_most_kernel(const void* W, int64_t K, int64_t N,
                                                             int64_t span,
                                                             uint32_t* most) {
  typedef typename elem<T>::storage S;
  constexpr int kCols = 16 / sizeof(S);
  typedef S V __attribute__((ext_vector_type(kCols), aligned(sizeof(S))));
  const int64_t e = blockIdx.z;
  const int64_t n = ((int64_t)blockIdx.x * kWave + lane_id()) * kCols;
  const int64_t k0 = (int64_t)blockIdx.y * span, k1 = k0 + span < K ? k0 + span : K;
  __shared__ uint32_t s_most[kThreads / kWave][kCols * kWave];
  const S* w = static_cast<const S*>(W) + e * K * N + n;
  uint32_t m[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) m[j] = 0;
  auto take = [&](int j, S v) {
    const uint32_t b = abs_bits(elem<T>::load(v));
    m[j] = b > m[j] ? b : m[j];
  };
  if (n + kCols <= N) {
#pragma unroll 16
    for (int64_t k = k0 + threadIdx.x / kWave; k < k1; k += kThreads / kWave) {
      const V v = *reinterpret_cast<const V*>(w + k * N);
#pragma unroll
      for (int j = 0; j < kCols; ++j) take(j, v[j]);
    }
  } else if (n < N) {
    for (int64_t k = k0 + threadIdx.x / kWave; k < k1; k += kThreads / kWave)
#pragma unroll
      for (int j = 0; j < kCols; ++j)
        if (n + j < N) take(j, w[k * N + j]);
  }
  // the waves' maxima: one atomic a column of the workgroup
#pragma unroll
  for (int j = 0; j < kCols; ++j) s_most[threadIdx.x / kWave][j * kWave + lane_id()] = m[j];
  __syncthreads();
  for (int i = threadIdx.x; i < kCols * kWave; i += kThreads) {
    const int64_t col = ((int64_t)blockIdx.x * kWave + i % kWave) * kCols + i / kWave;
    uint32_t top = s_most[0][i];
#pragma unroll
    for (int u = 1; u < kThreads / kWave; ++u) top = s_most[u][i] > top ? s_most[u][i] : top;
    if (col < N) atomicMax(&most[e * N + col], top);
  }
}

// A thread turns 4 reduction rows of C columns, a workgroup 64 rows of 16 threads'
// columns. In LDS a column's 64 bytes are padded to 68: words of neighbouring columns
// lie in different banks.
constexpr int kTurnPitch = kInt8Block + 4;
template <int C>
struct Turn {
  static constexpr int kColumns = C, kCols = 16 * C, kGroups = kCols / kInt8Block, kBytes = kCols * kTurnPitch;
  // thread: columns col .. + C - 1 and rows row .. + 3 of values; piece (operand t, lane
  // (g, i)) of integers
  const int col = threadIdx.x % 16 * C, row = threadIdx.x / 16 * 4;
  const int t = threadIdx.x / kWave, g = threadIdx.x % kWave / 16, i = threadIdx.x % 16;
  __device__ __forceinline__ uint32_t* word(int8_t* turn, int j) const {
    return reinterpret_cast<uint32_t*>(turn + (col + j) * kTurnPitch + row);
  }
  __device__ __forceinline__ uint32_t* piece(int8_t* turn, int group) const {
    return reinterpret_cast<uint32_t*>(
        turn + (group * kInt8Block + 16 * (i / 4) + 4 * t + i % 4) * kTurnPitch + g * 16);
  }
};

constexpr int kRun = 4;  // blocks of a workgroup along the reduction, loaded at once

// 64 columns by 256 reduction rows to integers (8 x 4,096 x 14,336 in bf16: 280 us, 128
// by 128 300). Grid: column groups, runs of blocks, experts.
template <typename T>
__global__ void __launch_bounds__(kThreads) int8_weight_kernel(const void* W, int64_t K, int64_t N,
                                                               const uint32_t* most, int8_t* codes,
                                                               float* scales) {
  typedef typename elem<T>::storage S;
  constexpr int C = 4;
  typedef Turn<C> U;
  constexpr float kMagic = 12582912.f;  // see Some::codes
  __shared__ __attribute__((aligned(16))) int8_t s_turn[2][U::kBytes];
  const int64_t e = blockIdx.z, n0 = (int64_t)blockIdx.x * U::kCols;
  const int64_t blocks = int8_pitch(K) / kInt8Block, b0 = (int64_t)blockIdx.y * kRun;
  const U at;
  const S* w = static_cast<const S*>(W) + e * K * N;
  Some<T, C> v[kRun][4];
#pragma unroll
  for (int u = 0; u < kRun; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t k = (b0 + u) * kInt8Block + at.row + i;
      v[u][i].load(w + k * N, k < K ? n0 + at.col : N, N);  // zeros past the last row
    }
  float s[C], inv[C];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int64_t n = n0 + at.col + j;
    s[j] = int8_scale(n < N ? most[e * N + n] : 0u);
    inv[j] = int8_inverse(s[j]);
    if (blockIdx.y == 0 && at.row == 0 && n < N) scales[e * N + n] = s[j];
  }
  uint4* out = reinterpret_cast<uint4*>(
                   codes + ((e * int8_groups(N) + blockIdx.x) * blocks + b0) * 4096) +
               threadIdx.x;
#pragma unroll
  for (int u = 0; u < kRun; ++u) {
    if (b0 + u >= blocks) break;
    int8_t* turn = s_turn[u & 1];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      uint32_t sum[4];
      float off = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = elem<T>::load(v[u][i].v[j]), near = fmaf(x, inv[j], kMagic);
        off = fmaxf(off, fabsf(fmaf(kMagic - near, s[j], x)));
        sum[i] = __float_as_uint(near);
      }
      uint32_t word = __builtin_amdgcn_perm(__builtin_amdgcn_perm(sum[3], sum[2], 0x0c0c0400u),
                                            __builtin_amdgcn_perm(sum[1], sum[0], 0x0c0c0400u),
                                            0x05040100u);
      if (!(off < 0.5f * s[j]) || inv[j] == 0.f) {
        int q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q[i] = int8_code(elem<T>::load(v[u][i].v[j]), s[j], inv[j]);
        word = pack_bytes(q[0], q[1], q[2], q[3]);
      }
      *at.word(turn, j) = word;
    }
    __syncthreads();
    const uint32_t* p = at.piece(turn, 0);
    out[(int64_t)u * (4096 / 16)] = make_uint4(p[0], p[1], p[2], p[3]);
  }
}

// And back, 256 bytes of a row in columns (283 us, by 128 bytes 310) and a block of
// reduction rows a workgroup (four on end, loaded at once: 410).
template <typename T>
__global__ void __launch_bounds__(kThreads) int8_weight_decode_kernel(const int8_t* codes,
                                                                      const float* scales,
                                                                      int64_t K, int64_t N,
                                                                      void* W) {
  typedef typename elem<T>::storage S;
  typedef Turn<16 / (int)sizeof(S)> U;
  __shared__ __attribute__((aligned(16))) int8_t s_turn[U::kBytes];
  const int64_t e = blockIdx.z, groups = int8_groups(N), n0 = (int64_t)blockIdx.x * U::kCols;
  const int64_t k0 = (int64_t)blockIdx.y * kInt8Block, blocks = int8_pitch(K) / kInt8Block;
  const U at;
  uint4 q[U::kGroups];
#pragma unroll
  for (int h = 0; h < U::kGroups; ++h) {
    const int64_t group = (int64_t)blockIdx.x * U::kGroups + h;
    q[h] = reinterpret_cast<const uint4*>(
        codes + ((e * groups + (group < groups ? group : groups - 1)) * blocks + blockIdx.y) *
                    4096)[threadIdx.x];
  }
#pragma unroll
  for (int h = 0; h < U::kGroups; ++h) {
    uint32_t* p = at.piece(s_turn, h);
    p[0] = q[h].x, p[1] = q[h].y, p[2] = q[h].z, p[3] = q[h].w;
  }
  Some<float, U::kColumns> s;
  s.load(scales + e * N, n0 + at.col, N);
  __syncthreads();
  if (n0 + at.col >= N) return;
  Some<T, U::kColumns> v[4];
#pragma unroll
  for (int j = 0; j < U::kColumns; ++j) {
    const uint32_t word = *at.word(s_turn, j);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i].v[j] = int8_value<T>((int8_t)(word >> (8 * i)), s.v[j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t k = k0 + at.row + i;
    if (k < K) v[i].store(static_cast<S*>(W) + (e * K + k) * N, n0 + at.col, N);
  }
}

int check_rows(int dtype, int64_t rows, int64_t f) {
  if (!int8_float(dtype)) return NT_ERR_DTYPE;
  if (rows < 0 || f < 1) return NT_ERR_INVALID_ARG;
  if (rows > kInt8MaxRows || f > kInt8MaxK) return NT_ERR_TOO_LARGE;
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

size_t nt_int8_rows_bytes(int64_t rows, int64_t f) {
  return check_rows(NT_F32, rows, f) == NT_OK ? (size_t)int8_rows_bytes(rows, int8_pitch(f)) : 0;
}

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
    auto launch = [&](auto kernel, int at_once, int team) {
      const int64_t parts = 16 / at_once, blocks = ceil_div(ceil_div(rows, (int64_t)16), (int64_t)8);
      hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks * 8 * parts)), dim3(at_once * team), 0,
                         stream, x, rows, f, codes, scales);
    };
    auto one = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream, x, f, codes,
                         scales);
    };
    const int64_t chunks = int8_pitch(f) / kVec;
    if (rows <= 512) {
      if (chunks <= 256) one(int8_row_kernel<T, 1, true>);
      else if (chunks <= 512) one(int8_row_kernel<T, 2, true>);
      else if (chunks <= 1024) one(int8_row_kernel<T, 4, true>);
      else one(int8_row_kernel<T, 4, false>);
    } else if (chunks <= 16) launch(int8_rows_kernel<T, 8, 32, 1, true>, 8, 32);
    else if (chunks <= 32) launch(int8_rows_kernel<T, 8, 32, 2, true>, 8, 32);
    else if (chunks <= 64) launch(int8_rows_kernel<T, 8, 64, 2, true>, 8, 64);
    else if (chunks <= 128) launch(int8_rows_kernel<T, 8, 64, 4, true>, 8, 64);
    else if (chunks <= 256) launch(int8_rows_kernel<T, 4, 128, 4, true>, 4, 128);
    else if (chunks <= 512) launch(int8_rows_kernel<T, 4, 128, 8, true>, 4, 128);
    else if (chunks <= 1024) launch(int8_rows_kernel<T, 4, 256, 8, true>, 4, 256);
    else launch(int8_rows_kernel<T, 4, 256, 8, false>, 4, 256);
  });
  return launch_status();
}

int nt_int8_rows_decode(int dtype, const int8_t* codes, const float* scales, int64_t rows,
                        int64_t f, void* x, hipStream_t stream) {
  const int st = check_rows(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  if (x == nullptr || codes == nullptr || scales == nullptr || !aligned16(codes))
    return NT_ERR_INVALID_ARG;
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    hipLaunchKernelGGL((int8_rows_decode_kernel<T>),
                       dim3((unsigned)ceil_div(rows, (int64_t)16),
                            (unsigned)ceil_div(f, (int64_t)(kWave * kVec))),
                       dim3(kThreads), 0, stream, codes, scales, rows, f, x);
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
    // Long spans for few atomics (they run at memory, not in an XCD's L2), but four
    // workgroups a CU (both passes, 8 x 4,096 x 14,336 bf16: spans of 64 rows 551 us,
    // 512 469, 2,048 580; 16 x 512 x 2,048: 31 and 63).
    const int64_t cols = ceil_div(N * dtype_bytes(dtype), (int64_t)kMostBytes);
    int64_t span = 1024;
    while (span > 64 && E * cols * ceil_div(K, span) < 1024) span /= 2;
    hipLaunchKernelGGL((int8_most_kernel<T>),
                       dim3((unsigned)cols, (unsigned)ceil_div(K, span), (unsigned)E),
                       dim3(kThreads), 0, stream, W, K, N, span, most);
    hipLaunchKernelGGL((int8_weight_kernel<T>),
                       dim3((unsigned)int8_groups(N),
                            (unsigned)ceil_div(int8_pitch(K), (int64_t)(kRun * kInt8Block)),
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
                       dim3((unsigned)ceil_div(N, (int64_t)(256 / dtype_bytes(dtype))),
                            (unsigned)ceil_div(K, (int64_t)kInt8Block), (unsigned)E),
                       dim3(kThreads), 0, stream, codes, scales, K, N, W);
  });
  return launch_status();
}

}  // extern "C"
