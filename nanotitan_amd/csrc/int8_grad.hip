// Gradients through frozen 8-bit weights, for 16-bit activations:
//
//   dX[a, k] = sum_n dOut[a, n] w[e, n, k],   w = q s[e, n] rounded to the type
//
// on the 16-bit matrix cores. The weights are read as integers, a quarter of what
// bringing them to 16 bits first would read and write, and turned on the way to LDS:
// a thread's 64 bytes are 16 values of k for four neighbouring n, and it writes for
// each k its four n. (v + 128) s - 128 s as one fused multiply-add rounds q s once.
//
// The epilogues keep float32 up to their one rounding: the gradient of the hidden
// values is not rounded before the activation's gradient is taken of it.
#include <algorithm>
#include <type_traits>

#include "gemm_common.hpp"
#include "int8_gemm.hpp"

namespace nt {
namespace {

enum Int8GradEpilogue { kGradPlain = 0, kGradDual = 1, kGradGelu = 2, kGradSwiGLU = 3 };

struct Int8Grad {
  Int8Gemm rows;           // offsets, E, A; K: output columns, N: the reduction
  const void *dout, *dout2;  // [A, N]; of the second matrix
  const void *aux, *aux2;    // gelu' or gate, value [A, K]
};

constexpr int kGradBM = 128, kGradBN = 256, kGradWaves = 4;
constexpr int kGradThreads = kGradWaves * kWave;

// A row (a value of k) of the turned weights is 64 n, 8 chunks of 16 bytes; chunk c
// is stored at c ^ turned_swizzle(k). An operand takes rows 16 j + 4 t + m (j, m
// < 4), whose swizzles are all eight values twice: its reads touch every bank once.
__device__ __forceinline__ int turned_swizzle(int k) { return (k >> 1 & 1) | (k >> 4 & 3) << 1; }

template <typename T, int EPI>
__global__ void __launch_bounds__(kGradThreads, 2) int8_grad_kernel(Int8Grad g) {
  typedef typename elem<T>::storage S;
  typedef typename mfma_op<T>::vec vec;
  const Int8Gemm& a = g.rows;
  constexpr int BM = kGradBM, BN = kGradBN, WGN = 2;
  constexpr int AB = BM / 2 / 16, CG = BN / 2 / 64;  // of a wave: 64 rows by 128 columns
  typedef OperandTile<BM, true, 64, kGradWaves> TA;
  constexpr int kA = TA::kBytes, kB = BN * 128;
  __shared__ __attribute__((aligned(1024))) char smem[2 * kA + kB];
  __shared__ int32_t s_pref[NT_MAX_EXPERTS + 1];
  char* turned = smem + 2 * kA;
  int8_row_tiles(a, BM, s_pref);
  const int64_t total = (int64_t)__builtin_amdgcn_readfirstlane(s_pref[a.E]) * a.ntn;
  constexpr int kXcd = 8;
  const int64_t G = gridDim.x, wg = blockIdx.x;
  const int xcd = (int)(wg % kXcd);
  const int64_t q = G / kXcd, r = G % kXcd;
  const int64_t before = xcd * q + (xcd < r ? xcd : r);
  const int64_t nbx = q + (xcd < r ? 1 : 0);
  const int64_t t_end = __builtin_amdgcn_readfirstlane(
      (int)xcd_range_start(total, before + nbx, G, s_pref, a.E, a.ntn));
  const int64_t t_beg = __builtin_amdgcn_readfirstlane(
      (int)xcd_range_start(total, before, G, s_pref, a.E, a.ntn));

  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WGN, wn = wave % WGN;
  const int64_t kpitch = int8_pitch(a.K), kblocks = kpitch / kInt8Block;
  const int64_t groups = int8_groups(a.N);
  const int nk1 = (int)ceil_div(a.N, (int64_t)64), nk = EPI == kGradDual ? 2 * nk1 : nk1;
  TA ta;
  ta.init(a.N, wave, lane);
  FragReader<BM, true, AB, 64> fa;
  fa.init(wm * 64, lane);
  // thread: 16 values of k, four n from n0 on
  const int t4 = lane >> 4, g4 = lane >> 2 & 3, i4 = lane & 3, n0 = 16 * i4 + 4 * t4;

  for (int64_t logical = t_beg + wg / kXcd; logical < t_end; logical += nbx) {
    int e, nt;
    int64_t r0, r1, mtl;
    expert_tile_coords(logical, s_pref, a.E, a.ntn, e, mtl, nt);
    int8_expert_rows(a, e, r0, r1);
    e = __builtin_amdgcn_readfirstlane(e);
    nt = __builtin_amdgcn_readfirstlane(nt);
    const int64_t row0 = (int64_t)__builtin_amdgcn_readfirstlane((int)(r0 + mtl * BM));
    const int64_t left = (int64_t)__builtin_amdgcn_readfirstlane((int)r1) - row0;
    const int rows = (int)(left < BM ? left : BM);
    const int64_t col0 = (int64_t)nt * BN;
    // this wave turns one block of 64 columns (none past the last)
    const int64_t kb = col0 / kInt8Block + wave;
    const bool has = kb < kblocks;

    uint4 w[4];
    float4 s;
    auto fetch = [&](int kt, char* lds) {
      const bool second = EPI == kGradDual && kt >= nk1;
      const int64_t nb = second ? kt - nk1 : kt;
      const int8_t* m = second ? a.w2 : a.w;
      const float* sc = second ? a.w2_scales : a.w_scales;
      const int8_t* at = m + ((e * groups + nb) * kblocks + (has ? kb : kblocks - 1)) * 4096 +
                         lane * 64;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint4*>(at)[i];
      const int64_t n = nb * 64 + n0;
      s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (n < a.N) {  // (N is a multiple of 8)
        typedef float V4 __attribute__((ext_vector_type(4), aligned(4)));
        const V4 v = *reinterpret_cast<const V4*>(sc + e * a.N + n);
        s = make_float4(v[0], v[1], v[2], v[3]);
      }
      const int64_t kv = a.N - nb * 64 < 64 ? a.N - nb * 64 : 64;
      const S* d = static_cast<const S*>(second ? g.dout2 : g.dout) + row0 * a.N + nb * 64;
      ta.issue(d, ((rows - 1) * a.N + kv) * 2, lds, kv, wave);
    };
    auto turn = [&]() {
      const float sc[4] = {s.x, s.y, s.z, s.w};
      uint32_t u[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int d = 0; d < 4; ++d) u[i][d] = v[d] ^ 0x80808080u;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = fmaf((float)(u[i][j / 4] >> (8 * (j % 4)) & 255u), sc[i], -128.f * sc[i]);
        const int k = wave * 64 + 16 * g4 + j;
        *reinterpret_cast<uint2*>(turned + k * 128 +
                                  ((2 * i4 + (t4 >> 1)) ^ turned_swizzle(k)) * 16 +
                                  (t4 & 1) * 8) =
            make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
      }
    };

    f32x4_t acc[AB][CG][4];
#pragma unroll
    for (int b = 0; b < AB; ++b)
#pragma unroll
      for (int c = 0; c < CG; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[b][c][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    __syncthreads();  // the tile before is read no more
    fetch(0, smem);
    for (int kt = 0; kt < nk; ++kt) {
      wait_vmcnt<0>();  // this step's rows are in LDS, its weights in registers
      turn();
      __syncthreads();
      if (kt + 1 < nk) fetch(kt + 1, smem + (kt + 1 & 1) * kA);
      const char* sa = smem + (kt & 1) * kA;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        vec x[AB];
#pragma unroll
        for (int b = 0; b < AB; ++b) x[b] = fa.template read<vec>(sa, b, ks);
#pragma unroll
        for (int c = 0; c < CG; ++c)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int k = (wn * CG + c) * 64 + 16 * ((lane & 15) >> 2) + 4 * t + (lane & 3);
            const vec y = *reinterpret_cast<const vec*>(
                turned + k * 128 + ((4 * ks + (lane >> 4)) ^ turned_swizzle(k)) * 16);
#pragma unroll
            for (int b = 0; b < AB; ++b) acc[b][c][t] = mfma_op<T>::run(y, x[b], acc[b][c][t]);
          }
      }
      __syncthreads();
    }
    // lane: row l % 16 of a block, columns 16 (l / 16) .. + 15 of a group
#pragma unroll
    for (int c = 0; c < CG; ++c) {
      const int64_t n = col0 + (wn * CG + c) * 64 + 16 * (lane >> 4);
      const int width = (int)(a.K - n < 16 ? a.K - n : 16);
#pragma unroll
      for (int b = 0; b < AB; ++b) {
        const int m = wm * 64 + 16 * b + (lane & 15);
        if (m >= rows || n >= a.K) continue;
        const int64_t at = (row0 + m) * a.K + n;
        S o[3][16], x1[16], x2[16];
        if constexpr (EPI == kGradGelu || EPI == kGradSwiGLU) int8_get<T>(g.aux, at, width, x1);
        if constexpr (EPI == kGradSwiGLU) int8_get<T>(g.aux2, at, width, x2);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float d = acc[b][c][j / 4][j % 4];
          if constexpr (EPI == kGradGelu) {
            o[0][j] = to_bits<T>(d * elem<T>::load(x1[j]));
          } else if constexpr (EPI == kGradSwiGLU) {
            const float z = elem<T>::load(x1[j]), sg = sigmoid_of<T>(z);
            o[0][j] = to_bits<T>(d * elem<T>::load(x2[j]) * sg * (1.f + z * (1.f - sg)));
            o[1][j] = to_bits<T>(d * z * sg);
          } else {
            o[0][j] = to_bits<T>(d);
          }
        }
        int8_put<T, EPI == kGradSwiGLU ? 2 : 1>(a, at, width, o);
      }
    }
  }
}

int run_grad(int dtype, int epi, Int8Grad g, hipStream_t s) {
  Int8Gemm& a = g.rows;
  if (dtype != NT_F16 && dtype != NT_BF16) return NT_ERR_DTYPE;
  if (a.E < 1 || a.A < 0 || a.K < 1 || a.N < 1 || a.N % 8 != 0) return NT_ERR_INVALID_ARG;
  if (a.E > NT_MAX_EXPERTS) return NT_ERR_TOO_MANY_EXPERTS;
  if (a.K > kInt8MaxK || a.N > 1 << 20 || a.A > kInt8MaxRows) return NT_ERR_TOO_LARGE;
  if (a.A == 0) return NT_OK;
  auto bad = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  if (g.dout == nullptr || a.w == nullptr || a.w_scales == nullptr || a.out == nullptr ||
      (a.offsets == nullptr && a.E != 1) || bad(g.dout) || bad(a.w) ||
      (epi == kGradDual && (g.dout2 == nullptr || a.w2 == nullptr || a.w2_scales == nullptr ||
                            bad(g.dout2) || bad(a.w2))) ||
      (epi >= kGradGelu && g.aux == nullptr) ||
      (epi == kGradSwiGLU && (g.aux2 == nullptr || a.out2 == nullptr)))
    return NT_ERR_INVALID_ARG;
  a.ntn = (int32_t)ceil_div(a.K, (int64_t)kGradBN);
  const int64_t tiles = (ceil_div(a.A, (int64_t)kGradBM) + a.E - 1) * a.ntn;
  if (tiles > INT32_MAX) return NT_ERR_TOO_LARGE;
  const unsigned grid = (unsigned)std::min<int64_t>(tiles, 2 * (int64_t)device_cus(s));
  auto go = [&](auto type) {
    typedef typename decltype(type)::type T;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(grid), dim3(kGradThreads), 0, s, g);
    };
    if (epi == kGradPlain) launch(int8_grad_kernel<T, kGradPlain>);
    else if (epi == kGradDual) launch(int8_grad_kernel<T, kGradDual>);
    else if (epi == kGradGelu) launch(int8_grad_kernel<T, kGradGelu>);
    else launch(int8_grad_kernel<T, kGradSwiGLU>);
  };
  if (dtype == NT_F16) go(tag<f16>());
  else go(tag<bf16>());
  return launch_status();
}

Int8Grad make_grad(const int8_t* w, const float* w_scales, const int32_t* offsets,
                   const void* dout, int32_t E, int64_t A, int64_t K, int64_t N, void* out) {
  Int8Grad g = {};
  g.rows.w = w, g.rows.w_scales = w_scales, g.rows.offsets = offsets;
  g.rows.E = E, g.rows.A = A, g.rows.K = K, g.rows.N = N, g.rows.out = out;
  g.dout = dout;
  return g;
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int nt_int8_grouped_gemm_dx(int dtype, const int8_t* w, const float* w_scales,
                            const int32_t* offsets, const void* dout, int32_t E, int64_t A,
                            int64_t K, int64_t N, void* dx, hipStream_t stream) {
  return run_grad(dtype, kGradPlain, make_grad(w, w_scales, offsets, dout, E, A, K, N, dx),
                  stream);
}

int nt_int8_grouped_gemm_dx2(int dtype, const int8_t* w1, const float* scales1, const int8_t* w2,
                             const float* scales2, const int32_t* offsets, const void* dout1,
                             const void* dout2, int32_t E, int64_t A, int64_t K, int64_t N,
                             void* dx, hipStream_t stream) {
  Int8Grad g = make_grad(w1, scales1, offsets, dout1, E, A, K, N, dx);
  g.rows.w2 = w2, g.rows.w2_scales = scales2, g.dout2 = dout2;
  return run_grad(dtype, kGradDual, g, stream);
}

int nt_int8_grouped_gemm_dx_gelu(int dtype, const int8_t* w, const float* w_scales,
                                 const int32_t* offsets, const void* dout, const void* act_grad,
                                 int32_t E, int64_t A, int64_t K, int64_t N, void* dh,
                                 hipStream_t stream) {
  Int8Grad g = make_grad(w, w_scales, offsets, dout, E, A, K, N, dh);
  g.aux = act_grad;
  return run_grad(dtype, kGradGelu, g, stream);
}

int nt_int8_grouped_gemm_dx_swiglu(int dtype, const int8_t* w, const float* w_scales,
                                   const int32_t* offsets, const void* dout, const void* gate,
                                   const void* value, int32_t E, int64_t A, int64_t K, int64_t N,
                                   void* dgate, void* dvalue, hipStream_t stream) {
  Int8Grad g = make_grad(w, w_scales, offsets, dout, E, A, K, N, dgate);
  g.aux = gate, g.aux2 = value, g.rows.out2 = dvalue;
  return run_grad(dtype, kGradSwiGLU, g, stream);
}

}  // extern "C"
