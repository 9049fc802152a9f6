// Activation checkpoints in 8 bits and their use in the backward.
//
// 32 consecutive columns of a row share a power of two 2^x, x the least
// integer (>= -127) with max|v| < 127.5 2^x; a value is kept as the int8
// nearest to v 2^-x (ties to even) and the block as the byte x + 127. Scaling
// by a power of two is exact, so a value is off by half a unit at most: 2^-7
// of the block's largest value, 0.3 to 0.6 % of a normal block's deviation (an
// 8-bit float with 3 mantissa bits: 2.6 % of each value). Decoding is exact in
// every activation type: 7 bits fit bf16's 8. A block with an infinity or a NaN
// gets the byte 255 and decodes to NaN; a value that rounds past the type's
// largest decodes to that.
//
// The activation kernels read an expert FFN's pre-activations once, write its
// hidden values and the checkpoint; their backwards read the checkpoint and
// the hidden gradient, and write the pre-activations' gradients and, for the
// down projection's weight gradient, the hidden values again. All of it is
// bound by HBM; a lane holds eight columns, four lanes a block.
#include <algorithm>

#include "common.hpp"

namespace nt {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;
constexpr int kBlock = 32;
constexpr int kLanes = kBlock / kVec;  // lanes of a block

__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  // over the four lanes of a quad: lane ^ 1, then lane ^ 2
  const uint32_t a = __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);
  v = v > a ? v : a;
  const uint32_t b = __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);
  return v > b ? v : b;
}

// The shared exponent's byte from the bits of max|v|.
__device__ __forceinline__ uint32_t block_byte(uint32_t most) {
  if (most >= 0x7f800000u) return 255u;
  const int x = (int)(most >> 23) - 6 + ((most & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
  return x < 0 ? 0u : (uint32_t)x;
}
// 2^-x and 2^x of a byte x + 127 (at most 249 for finite blocks).
__device__ __forceinline__ float down_scale(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float up_scale(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x400000u : byte << 23);
}

// A wave's place: the row and chunk (eight columns) of each lane. Chunks per
// row are a multiple of four, so that a block's lanes are one quad; rows are
// counted in 64 bits per workgroup and in 32 inside it.
struct Place {
  int64_t row;
  int32_t c0;
  bool live;
};
__device__ __forceinline__ Place place(int64_t rows, int32_t chunks, int64_t item) {
  Place p;
  p.row = item / chunks;
  p.c0 = (int32_t)(item - p.row * chunks) * kVec;
  p.live = p.row < rows;
  return p;
}

template <typename T>
__device__ __forceinline__ void load8(const typename elem<T>::storage* p, int64_t row, int32_t c0,
                                      int32_t f, bool live, float (&v)[kVec]) {
  typename elem<T>::storage s[kVec];
  if (live && c0 + kVec <= f) {
    __builtin_memcpy(s, p + row * f + c0, sizeof(s));
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = elem<T>::load(s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      v[i] = live && c0 + i < f ? elem<T>::load(p[row * f + c0 + i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(typename elem<T>::storage* p, int64_t row, int32_t c0,
                                       int32_t f, bool live, const float (&v)[kVec]) {
  typename elem<T>::storage s[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) s[i] = elem<T>::store(v[i]);
  if (live && c0 + kVec <= f) {
    __builtin_memcpy(p + row * f + c0, s, sizeof(s));
  } else if (live) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (c0 + i < f) p[row * f + c0 + i] = s[i];
  }
}

// The checkpoint of the lane's eight values (zeros past the row's end).
__device__ __forceinline__ void keep8(const float (&v)[kVec], int8_t* codes, uint8_t* bytes,
                                      int64_t row, int32_t c0, int32_t f, int32_t chunks,
                                      bool live) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    most = b > most ? b : most;
  }
  const uint32_t byte = block_byte(dpp_max(most));
  const float s = down_scale(byte);
  int8_t q[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) q[i] = byte == 255u ? 0 : (int8_t)(int)rintf(v[i] * s);
  if (!live) return;
  if (c0 + kVec <= f) {
    __builtin_memcpy(codes + row * f + c0, q, sizeof(q));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (c0 + i < f) codes[row * f + c0 + i] = q[i];
  }
  if ((lane_id() & (kLanes - 1)) == 0) bytes[row * (chunks / kLanes) + c0 / kBlock] = (uint8_t)byte;
}

// The largest finite value of T, and the byte of the blocks that can round past
// it: 64 units, next to the largest value, are a power of two out of range.
template <typename T>
struct range {
  static constexpr uint32_t most = sizeof(typename elem<T>::storage) == 4 ? 0x7f7fffffu : 0x7f7f0000u;
  static constexpr uint32_t byte = 249;
};
template <>
struct range<f16> {
  static constexpr uint32_t most = 0x477fe000u;  // 65504
  static constexpr uint32_t byte = 137;
};

template <typename T>
__device__ __forceinline__ void held8(const int8_t* codes, const uint8_t* bytes, int64_t row,
                                      int32_t c0, int32_t f, int32_t chunks, bool live,
                                      float (&v)[kVec]) {
  int8_t q[kVec];
  if (live && c0 + kVec <= f) {
    __builtin_memcpy(q, codes + row * f + c0, sizeof(q));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) q[i] = live && c0 + i < f ? codes[row * f + c0 + i] : 0;
  }
  const uint32_t byte = live ? bytes[row * (chunks / kLanes) + c0 / kBlock] : 0u;
  const float s = up_scale(byte);
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i] = (float)q[i] * s;
  if (byte >= range<T>::byte) {
    const float most = __uint_as_float(range<T>::most);
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = v[i] > most ? most : v[i] < -most ? -most : v[i];  // NaN stays
  }
}

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

struct Act8Args {
  const void *a, *b;        // pre-activation (gate), value; backward: the hidden gradient in a
  void *out, *da, *db;      // hidden; backward: gradients
  int8_t *qa, *qb;
  uint8_t *xa, *xb;
  int64_t rows;
  int32_t f, chunks;
};

enum { kCopy8 = 0, kGelu8 = 1, kSwiGLU8 = 2 };

// Forward: out = act(a[, b]) (kCopy8: none) and the checkpoints of a and b.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) keep8_kernel(Act8Args g) {
  typedef typename elem<T>::storage S;
  const Place p = place(g.rows, g.chunks, (int64_t)blockIdx.x * kThreads + threadIdx.x);
  float a[kVec], b[kVec], o[kVec];
  load8<T>(static_cast<const S*>(g.a), p.row, p.c0, g.f, p.live, a);
  if constexpr (ACT == kSwiGLU8) load8<T>(static_cast<const S*>(g.b), p.row, p.c0, g.f, p.live, b);
  if constexpr (ACT != kCopy8) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      o[i] = ACT == kSwiGLU8 ? a[i] * sigmoid(a[i]) * b[i]
                             : 0.5f * a[i] * (1.f + erff(a[i] * 0.70710678f));
    store8<T>(static_cast<S*>(g.out), p.row, p.c0, g.f, p.live, o);
  }
  if (g.qa == nullptr) return;  // the activation alone
  keep8(a, g.qa, g.xa, p.row, p.c0, g.f, g.chunks, p.live);
  if constexpr (ACT == kSwiGLU8) keep8(b, g.qb, g.xb, p.row, p.c0, g.f, g.chunks, p.live);
}

// Backward at the checkpoint's values: da (and db) from the hidden gradient
// in a, and the hidden values again where out is wanted. kCopy8: decode to out.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) held8_kernel(Act8Args g) {
  typedef typename elem<T>::storage S;
  const Place p = place(g.rows, g.chunks, (int64_t)blockIdx.x * kThreads + threadIdx.x);
  float a[kVec], b[kVec], d[kVec], o[kVec];
  held8<T>(g.qa, g.xa, p.row, p.c0, g.f, g.chunks, p.live, a);
  if constexpr (ACT == kCopy8) {
    store8<T>(static_cast<S*>(g.out), p.row, p.c0, g.f, p.live, a);
    return;
  }
  load8<T>(static_cast<const S*>(g.a), p.row, p.c0, g.f, p.live, d);
  if constexpr (ACT == kSwiGLU8) {
    held8<T>(g.qb, g.xb, p.row, p.c0, g.f, g.chunks, p.live, b);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float s = sigmoid(a[i]), silu = a[i] * s;
      o[i] = silu * b[i];
      b[i] *= d[i] * s * (1.f + a[i] * (1.f - s));  // the gate's gradient
      d[i] *= silu;                                 // the value's
    }
    store8<T>(static_cast<S*>(g.da), p.row, p.c0, g.f, p.live, b);
    store8<T>(static_cast<S*>(g.db), p.row, p.c0, g.f, p.live, d);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float cdf = 0.5f * (1.f + erff(a[i] * 0.70710678f));
      const float pdf = __expf(-0.5f * a[i] * a[i]) * 0.39894228f;
      o[i] = a[i] * cdf;
      d[i] *= cdf + a[i] * pdf;
    }
    store8<T>(static_cast<S*>(g.da), p.row, p.c0, g.f, p.live, d);
  }
  if (g.out != nullptr) store8<T>(static_cast<S*>(g.out), p.row, p.c0, g.f, p.live, o);
}

int check8(int dtype, int64_t rows, int64_t f) {
  if (dtype != NT_F32 && dtype != NT_F16 && dtype != NT_BF16) return NT_ERR_DTYPE;
  if (rows < 0 || f < 1) return NT_ERR_INVALID_ARG;
  if (f > (1 << 30) || rows > INT32_MAX) return NT_ERR_TOO_LARGE;
  // workgroups of 256 chunks
  if (rows * (ceil_div(f, kBlock) * kLanes) > (int64_t)INT32_MAX * kThreads)
    return NT_ERR_TOO_LARGE;
  return NT_OK;
}

template <int ACT, bool FORWARD>
int launch8(int dtype, Act8Args g, hipStream_t stream) {
  g.chunks = (int32_t)(ceil_div(g.f, kBlock) * kLanes);
  const dim3 grid((unsigned)ceil_div(g.rows * g.chunks, (int64_t)kThreads));
  auto run = [&](auto t) {
    if constexpr (FORWARD)
      hipLaunchKernelGGL((keep8_kernel<decltype(t), ACT>), grid, dim3(kThreads), 0, stream, g);
    else
      hipLaunchKernelGGL((held8_kernel<decltype(t), ACT>), grid, dim3(kThreads), 0, stream, g);
  };
  if (dtype == NT_F32) run(float());
  else if (dtype == NT_F16) run(f16());
  else run(bf16());
  return launch_status();
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int64_t nt_checkpoint8_blocks(int64_t f) { return f < 1 ? 0 : ceil_div(f, kBlock); }

int nt_checkpoint8(int dtype, const void* x, int64_t rows, int64_t f, int8_t* codes,
                   uint8_t* exps, hipStream_t stream) {
  const int st = check8(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  if (x == nullptr || codes == nullptr || exps == nullptr) return NT_ERR_INVALID_ARG;
  Act8Args g = {};
  g.a = x, g.qa = codes, g.xa = exps, g.rows = rows, g.f = (int32_t)f;
  return launch8<kCopy8, true>(dtype, g, stream);
}

int nt_checkpoint8_decode(int dtype, const int8_t* codes, const uint8_t* exps, int64_t rows,
                          int64_t f, void* x, hipStream_t stream) {
  const int st = check8(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  if (x == nullptr || codes == nullptr || exps == nullptr) return NT_ERR_INVALID_ARG;
  Act8Args g = {};
  g.out = x, g.qa = const_cast<int8_t*>(codes), g.xa = const_cast<uint8_t*>(exps);
  g.rows = rows, g.f = (int32_t)f;
  return launch8<kCopy8, false>(dtype, g, stream);
}

int nt_gelu_checkpoint8(int dtype, const void* h, int64_t rows, int64_t f, void* act,
                        int8_t* codes, uint8_t* exps, hipStream_t stream) {
  const int st = check8(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  if (h == nullptr || act == nullptr || (codes == nullptr) != (exps == nullptr))
    return NT_ERR_INVALID_ARG;
  Act8Args g = {};
  g.a = h, g.out = act, g.qa = codes, g.xa = exps, g.rows = rows, g.f = (int32_t)f;
  return launch8<kGelu8, true>(dtype, g, stream);
}

int nt_gelu_backward8(int dtype, const void* dact, const int8_t* codes, const uint8_t* exps,
                      int64_t rows, int64_t f, void* dh, void* act, hipStream_t stream) {
  const int st = check8(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  if (dact == nullptr || dh == nullptr || codes == nullptr || exps == nullptr)
    return NT_ERR_INVALID_ARG;
  Act8Args g = {};
  g.a = dact, g.out = act, g.da = dh, g.qa = const_cast<int8_t*>(codes);
  g.xa = const_cast<uint8_t*>(exps), g.rows = rows, g.f = (int32_t)f;
  return launch8<kGelu8, false>(dtype, g, stream);
}

int nt_swiglu_checkpoint8(int dtype, const void* gate, const void* value, int64_t rows, int64_t f,
                          void* hidden, int8_t* gate_codes, uint8_t* gate_exps,
                          int8_t* value_codes, uint8_t* value_exps, hipStream_t stream) {
  const int st = check8(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  const int kept = (gate_codes != nullptr) + (gate_exps != nullptr) + (value_codes != nullptr) +
                   (value_exps != nullptr);
  if (gate == nullptr || value == nullptr || hidden == nullptr || (kept != 0 && kept != 4))
    return NT_ERR_INVALID_ARG;
  Act8Args g = {};
  g.a = gate, g.b = value, g.out = hidden, g.qa = gate_codes, g.xa = gate_exps;
  g.qb = value_codes, g.xb = value_exps, g.rows = rows, g.f = (int32_t)f;
  return launch8<kSwiGLU8, true>(dtype, g, stream);
}

int nt_swiglu_backward8(int dtype, const void* dhidden, const int8_t* gate_codes,
                        const uint8_t* gate_exps, const int8_t* value_codes,
                        const uint8_t* value_exps, int64_t rows, int64_t f, void* dgate,
                        void* dvalue, void* hidden, hipStream_t stream) {
  const int st = check8(dtype, rows, f);
  if (st != NT_OK || rows == 0) return st;
  if (dhidden == nullptr || dgate == nullptr || dvalue == nullptr || gate_codes == nullptr ||
      gate_exps == nullptr || value_codes == nullptr || value_exps == nullptr)
    return NT_ERR_INVALID_ARG;
  Act8Args g = {};
  g.a = dhidden, g.out = hidden, g.da = dgate, g.db = dvalue;
  g.qa = const_cast<int8_t*>(gate_codes), g.xa = const_cast<uint8_t*>(gate_exps);
  g.qb = const_cast<int8_t*>(value_codes), g.xb = const_cast<uint8_t*>(value_exps);
  g.rows = rows, g.f = (int32_t)f;
  return launch8<kSwiGLU8, false>(dtype, g, stream);
}

}  // extern "C"
