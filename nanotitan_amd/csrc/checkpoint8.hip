// Activation checkpoints in 8 bits and their use in the backward.
//
// 32 consecutive columns of a row share a power of two 2^x, x the least
// integer (>= -127) with max|v| < 127.5 2^x; a value is kept as the int8
// nearest to v 2^-x (ties to even) and the block as the byte x + 127. Scaling
// by a power of two is exact, so a value is off by half a unit at most: 1/127.5
// of the block's largest value, as a norm 0.5 to 1.1 % of a normal block (an
// 8-bit float with 3 mantissa bits: 2.6 %). Decoding is exact in
// every activation type: 7 bits fit bf16's 8. A block with an infinity or a NaN
// gets the byte 255 and decodes to NaN; a value that rounds past the type's
// largest decodes to that.
//
// The activation kernels read an expert FFN's pre-activations once, write its
// hidden values and the checkpoint; their backwards read the checkpoint and
// the hidden gradient, and write the pre-activations' gradients and, for the
// down projection's weight gradient, the hidden values again. HBM bounds all
// of it as long as the arithmetic stays near 30 instructions a value, which is
// why the division and the conversions are written out below, and why 16-bit
// values take the fit of erfc that the plain path's epilogue takes (gelu.hpp).
//
// Measured on MI355X (a copy: 5.65 TB/s): SwiGLU of 61,440 x 2,048 bf16 187 us
// forward, 186 backward (5.45 TB/s); GELU of the same 115 (5.5) and 142 (4.5: with
// three quarter-rate instructions a value the vector units bound it); GELU of
// 10,007 x 1,365 fp16 19 and 26, of 1,344 columns, whose rows are aligned, 13 and
// 23% less.
#include <algorithm>

#include "bits.hpp"
#include "common.hpp"
#include "gelu.hpp"

namespace nt {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 16;  // columns of a lane: 16 bytes of codes
constexpr int kBlock = 32;
constexpr int kLanes = kBlock / kVec;  // lanes of a block

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

// A lane's row and its first column. Chunks per row are a multiple of two, so
// that a block's lanes are neighbours. The workgroup's first row is 64-bit and
// the same for all its lanes; from there on 32 bits do.
struct Place {
  int64_t row;
  int32_t c0;
  bool live;
};
__device__ __forceinline__ Place place(int64_t rows, int32_t chunks) {
  const int64_t first = (int64_t)blockIdx.x * kThreads, row0 = first / chunks;
  const uint32_t at = (uint32_t)(first - row0 * chunks) + threadIdx.x;
  const uint32_t down = at / (uint32_t)chunks;
  Place p;
  p.row = row0 + down;
  p.c0 = (int32_t)(at - down * (uint32_t)chunks) * kVec;
  p.live = p.row < rows;
  return p;
}

// A lane's sixteen values as they are stored, zeros past the row's end.
template <typename T>
struct Values {
  typedef typename elem<T>::storage S;
  typedef S V __attribute__((ext_vector_type(kVec), aligned(sizeof(S))));
  V v;
  __device__ __forceinline__ void load(const void* rows, const Place& p, int32_t f) {
    const S* at = static_cast<const S*>(rows) + p.row * f + p.c0;
    if (p.live && p.c0 + kVec <= f) {
      v = __builtin_nontemporal_load(reinterpret_cast<const V*>(at));
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = p.live && p.c0 + i < f ? at[i] : S(0);
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return elem<T>::load(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = to_bits<T>(x); }
  __device__ __forceinline__ void store(void* rows, const Place& p, int32_t f) const {
    S* at = static_cast<S*>(rows) + p.row * f + p.c0;
    if (p.live && p.c0 + kVec <= f) {
      *reinterpret_cast<V*>(at) = v;
    } else if (p.live) {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (p.c0 + i < f) at[i] = v[i];
    }
  }
  // Bits of the largest magnitude as a float; an infinity or a NaN is above
  // all others. 16-bit values are compared as pairs of integers.
  __device__ __forceinline__ uint32_t most() const {
    if constexpr (sizeof(S) == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
        m = b > m ? b : m;
      }
      return m;
    } else {
      typedef uint16_t U2 __attribute__((ext_vector_type(2)));
      U2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < kVec; i += 2) {
        const U2 b = U2{v[i], v[i + 1]} & U2{0x7fff, 0x7fff};
        m = __builtin_elementwise_max(m, b);
      }
      return __float_as_uint(elem<T>::load(m[0] > m[1] ? m[0] : m[1]));
    }
  }
};

typedef uint32_t Codes __attribute__((ext_vector_type(kVec / 4), aligned(1)));

// The checkpoint of the lane's values. Adding 1.5 * 2^23 rounds v 2^-x to an
// integer (ties to even) and leaves it in the sum's low byte.
template <typename T>
__device__ __forceinline__ void keep8(const Values<T>& v, int8_t* codes, uint8_t* bytes,
                                      const Place& p, int32_t f, int32_t chunks) {
  uint32_t most = v.most();
  const uint32_t other = __builtin_amdgcn_mov_dpp(most, 0xB1, 0xF, 0xF, true);  // lane ^ 1
  most = most > other ? most : other;
  const uint32_t byte = block_byte(most);
  const float s = down_scale(byte);
  Codes q;
#pragma unroll
  for (int i = 0; i < kVec / 4; ++i) {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(fmaf(v[i * 4 + j], s, 12582912.f));
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    q[i] = byte == 255u ? 0u : lo | hi;
  }
  if (!p.live) return;
  int8_t* at = codes + p.row * f + p.c0;
  if (p.c0 + kVec <= f) {
    *reinterpret_cast<Codes*>(at) = q;
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (p.c0 + i < f) at[i] = (int8_t)(q[i / 4] >> (8 * (i % 4)));
  }
  if ((lane_id() & (kLanes - 1)) == 0)
    bytes[p.row * (chunks / kLanes) + p.c0 / kBlock] = (uint8_t)byte;
}

// The largest finite value of T, and the byte from which a block can round past
// it (64 units, next to the largest value, are a power of two out of range) or
// 128 of its units pass float32's.
template <typename T>
struct range {
  static constexpr uint32_t most =
      sizeof(typename elem<T>::storage) == 4 ? 0x7f7fffffu : 0x7f7f0000u;
  static constexpr uint32_t byte = 248;
};
template <>
struct range<f16> {
  static constexpr uint32_t most = 0x477fe000u;  // 65504
  static constexpr uint32_t byte = 137;
};

// What a checkpoint holds: with the sign bit flipped a code is an unsigned
// byte, 128 above, which one instruction turns into a float.
struct Held {
  Codes q;
  uint32_t byte;
  __device__ __forceinline__ void load(const int8_t* codes, const uint8_t* bytes, const Place& p,
                                       int32_t f, int32_t chunks) {
    const int8_t* at = codes + p.row * f + p.c0;
    if (p.live && p.c0 + kVec <= f) {
      q = __builtin_nontemporal_load(reinterpret_cast<const Codes*>(at));
    } else {
#pragma unroll
      for (int i = 0; i < kVec / 4; ++i) q[i] = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (p.live && p.c0 + i < f) q[i / 4] |= (uint32_t)(uint8_t)at[i] << (8 * (i % 4));
    }
    byte = p.live ? bytes[p.row * (chunks / kLanes) + p.c0 / kBlock] : 0u;
  }
  template <typename T>
  __device__ __forceinline__ void values(float (&v)[kVec]) const {
    const float s = up_scale(byte), off = -128.f * s;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const uint32_t w = q[i / 4] ^ 0x80808080u;
      v[i] = fmaf((float)((w >> (8 * (i % 4))) & 0xffu), s, off);
    }
    if (byte >= range<T>::byte) {
      const float most = __uint_as_float(range<T>::most);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float x = (float)(int8_t)(q[i / 4] >> (8 * (i % 4))) * s;
        v[i] = x > most ? most : x < -most ? -most : x;  // NaN stays
      }
    }
  }
};

// 1 / (1 + e^-x): the reciprocal is within an ulp, the exponential's argument
// within half an ulp of x.
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-x));
}

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
  const Place p = place(g.rows, g.chunks);
  Values<T> a, b, o;
  a.load(g.a, p, g.f);
  if constexpr (ACT == kSwiGLU8) b.load(g.b, p, g.f);
  if constexpr (ACT != kCopy8) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      float bell;
      o.set(i, ACT == kSwiGLU8 ? a[i] * sigmoid(a[i]) * b[i] : a[i] * gelu_cdf<T>(a[i], bell));
    }
    o.store(g.out, p, g.f);
  }
  if (g.qa == nullptr) return;  // the activation alone
  keep8<T>(a, g.qa, g.xa, p, g.f, g.chunks);
  if constexpr (ACT == kSwiGLU8) keep8<T>(b, g.qb, g.xb, p, g.f, g.chunks);
}

// Backward at the checkpoint's values: da (and db) from the hidden gradient
// in a, and the hidden values again where out is wanted. kCopy8: decode to out.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) held8_kernel(Act8Args g) {
  const Place p = place(g.rows, g.chunks);
  Held ha, hb;
  ha.load(g.qa, g.xa, p, g.f, g.chunks);
  if constexpr (ACT == kSwiGLU8) hb.load(g.qb, g.xb, p, g.f, g.chunks);
  float a[kVec], b[kVec];
  if constexpr (ACT == kCopy8) {
    Values<T> x;
    ha.values<T>(a);
#pragma unroll
    for (int i = 0; i < kVec; ++i) x.set(i, a[i]);
    x.store(g.out, p, g.f);
    return;
  }
  Values<T> d, da, db, o;
  d.load(g.a, p, g.f);
  ha.values<T>(a);
  if constexpr (ACT == kSwiGLU8) {
    hb.values<T>(b);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float s = sigmoid(a[i]), silu = a[i] * s;
      o.set(i, silu * b[i]);
      da.set(i, d[i] * b[i] * fmaf(silu, 1.f - s, s));  // silu' = s + silu (1 - s)
      db.set(i, d[i] * silu);
    }
    db.store(g.db, p, g.f);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      float bell;
      const float cdf = gelu_cdf<T>(a[i], bell);
      o.set(i, a[i] * cdf);
      da.set(i, d[i] * fmaf(a[i] * 0.39894228f, bell, cdf));
    }
  }
  da.store(g.da, p, g.f);
  if (g.out != nullptr) o.store(g.out, p, g.f);
}

int check8(int dtype, int64_t rows, int64_t f) {
  if (dtype != NT_F32 && dtype != NT_F16 && dtype != NT_BF16) return NT_ERR_DTYPE;
  if (rows < 0 || f < 1) return NT_ERR_INVALID_ARG;
  if (f > (1 << 30) || rows > INT32_MAX) return NT_ERR_TOO_LARGE;
  // a thread for every chunk, in whole workgroups: a launch takes fewer than 2^32
  if (rows * (ceil_div(f, kBlock) * kLanes) > (int64_t)UINT32_MAX + 1 - kThreads)
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
