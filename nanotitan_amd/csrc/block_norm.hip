// Norms before and after a block, fused with the block's gate and residual
// scale, forward and backward.
//
//   N(v) = (v - m) r w + b   rms:   m = 0,       r = rsqrt(mean v^2 + eps)
//                            layer: m = mean v,  r = rsqrt(mean (v - m)^2 + eps)
//   p = N(y; w, b)  (p = y without a weight),  h = x + s g p rounded to x's
//   type,  n = N(h; w', b') of h as it is held.
// Backward, with D = dh + dN(dn; h, w') and dN(u) = r (u - [mean u] - vhat
// mean(u vhat)) for u = d w, vhat = (v - m) r, [.] for layer norms:
//   dx = D,  dp = D s g,  dy = dN(dp; y, w),  dg = D s p,  ds = sum_t D g p,
//   dw = sum_t dp yhat,  db = sum_t dp,  dw' = sum_t dn hhat,  db' = sum_t dn.
//
// All of it is bound by HBM: one pass over each row, its values held in
// registers (eight a thread) between the sums over the row and their use.
#include <algorithm>

#include "common.hpp"

namespace nt {
namespace {

constexpr int kVec = 8;               // columns of a thread's chunk
constexpr int kMaxThreads = 1024;
constexpr int64_t kMaxNormWidth = 2 * kMaxThreads * kVec;

// A row of up to a wave's threads shares its workgroup with others; a wider
// one has it alone.
constexpr int norm_threads(int row_threads) { return row_threads <= kWave ? 256 : row_threads; }

// Parameters (weights, biases, scale) come in one type of their own, read or
// written once per thread: a uniform branch on the type, no instantiations.
__device__ __forceinline__ float load_param(const void* p, int dt, int64_t i) {
  if (dt == NT_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return dt == NT_BF16 ? bf16_to_f32(v) : f16_to_f32(v);
}
__device__ __forceinline__ void store_param(void* p, int dt, int64_t i, float v) {
  if (dt == NT_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = dt == NT_BF16 ? f32_to_bf16(v) : f32_to_f16(v);
}

// A thread's chunk of a row: columns c0 .. c0 + 7 of d, zeros past the end.
// Rows of odd widths start at any element: the copies assume no alignment
// beyond the element's.
template <typename T>
__device__ __forceinline__ void load_chunk(const typename elem<T>::storage* row, int64_t c0,
                                           int64_t d, float (&v)[kVec]) {
  typename elem<T>::storage s[kVec];
  if (c0 + kVec <= d) {
    __builtin_memcpy(s, row + c0, sizeof(s));
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = elem<T>::load(s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = c0 + i < d ? elem<T>::load(row[c0 + i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_chunk(typename elem<T>::storage* row, int64_t c0, int64_t d,
                                            const float (&v)[kVec]) {
  typename elem<T>::storage s[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) s[i] = elem<T>::store(v[i]);
  if (c0 + kVec <= d) {
    __builtin_memcpy(row + c0, s, sizeof(s));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (c0 + i < d) row[c0 + i] = s[i];
  }
}
__device__ __forceinline__ void load_param_chunk(const void* p, int dt, int64_t c0, int64_t d,
                                                 float none, float (&v)[kVec]) {
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    v[i] = p == nullptr ? none : c0 + i < d ? load_param(p, dt, c0 + i) : 0.f;
}

// Sums over the TPR threads of a row, every thread receiving them: shuffles
// inside a wave, then LDS across the row's waves (one row per workgroup
// there). `s_red` holds N words a wave; calls alternate between two halves,
// so one barrier each is enough.
template <int TPR, int N>
struct RowSum {
  float* s_red;  // [2][N][waves]
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

struct NormArgs {
  const void *x, *y, *w, *b, *gate, *scale, *w_next, *b_next;
  void *h, *n;
  float* stats;  // [T][4]: mean and r of y, mean and r of h (may be null)
  int64_t T, d;
  float eps;
  int32_t param, gate_cols, scale_cols;
};

// mean and r of a row held in v (zeros past the width).
template <int TPR, int CH, bool LAYER, typename Sum>
__device__ __forceinline__ void row_stats(const float (&v)[CH][kVec], int64_t c0, int64_t d,
                                          float eps, Sum& sum, float& mean, float& r) {
  mean = 0.f;
  if constexpr (LAYER) {
    float t[1] = {0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < kVec; ++i) t[0] += v[c][i];
    sum(t);
    mean = t[0] / (float)d;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float u = v[c][i] - mean;
      if (!LAYER || c0 + c * TPR * kVec + i < d) q[0] = fmaf(u, u, q[0]);
    }
  sum(q);
  // the division and the root once a row: full precision costs nothing here
  r = 1.f / sqrtf(q[0] / (float)d + eps);
}

// One row per TPR threads, CH chunks of eight columns a thread (a row's
// chunks interleaved over its threads: coalesced 16-byte accesses).
template <typename TX, typename T, int TPR, int CH, bool LAYER>
__global__ void __launch_bounds__(norm_threads(TPR))
block_norm_kernel(NormArgs a) {
  typedef typename elem<TX>::storage SX;
  typedef typename elem<T>::storage S;
  constexpr int kThreads = norm_threads(TPR);
  constexpr int kRows = kThreads / TPR;
  __shared__ float s_red[2 * (kThreads / kWave)];
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  if (TPR <= kWave ? row >= a.T : false) return;  // wider rows: one a workgroup, all live
  const int64_t c0 = (int64_t)(threadIdx.x % TPR) * kVec, d = a.d, base = row * d;
  RowSum<TPR, 1> sum{s_red};
  float h[CH][kVec], p[CH][kVec];
  float mean_y = 0.f, r_y = 1.f, mean_h = 0.f, r_h = 1.f;
  const SX* x = static_cast<const SX*>(a.x) + base;
#pragma unroll
  for (int c = 0; c < CH; ++c) load_chunk<TX>(x, c0 + c * TPR * kVec, d, h[c]);
  if (a.y != nullptr) {
    const S* y = static_cast<const S*>(a.y) + base;
#pragma unroll
    for (int c = 0; c < CH; ++c) load_chunk<T>(y, c0 + c * TPR * kVec, d, p[c]);
    if (a.w != nullptr) row_stats<TPR, CH, LAYER>(p, c0, d, a.eps, sum, mean_y, r_y);
    const float g_row = a.gate != nullptr && a.gate_cols == 1
                            ? elem<T>::load(static_cast<const S*>(a.gate)[row]) : 1.f;
    const float s_all = a.scale != nullptr && a.scale_cols == 1 ? load_param(a.scale, a.param, 0)
                                                               : 1.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t cc = c0 + c * TPR * kVec;
      float w[kVec], b[kVec], g[kVec], sc[kVec];
      load_param_chunk(a.w, a.param, cc, d, 1.f, w);
      load_param_chunk(a.b, a.param, cc, d, 0.f, b);
      load_param_chunk(a.scale_cols == 1 ? nullptr : a.scale, a.param, cc, d, s_all, sc);
      if (a.gate != nullptr && a.gate_cols != 1) {
        load_chunk<T>(static_cast<const S*>(a.gate) + base, cc, d, g);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) g[i] = g_row;
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float v = fmaf((p[c][i] - mean_y) * r_y, w[i], b[i]);
        h[c][i] = elem<TX>::load(elem<TX>::store(fmaf(sc[i] * g[i], v, h[c][i])));
        if (cc + i >= d) h[c][i] = 0.f;
      }
      store_chunk<TX>(static_cast<SX*>(a.h) + base, cc, d, h[c]);
    }
  }
  if (a.w_next != nullptr) {
    row_stats<TPR, CH, LAYER>(h, c0, d, a.eps, sum, mean_h, r_h);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t cc = c0 + c * TPR * kVec;
      float w[kVec], b[kVec];
      load_param_chunk(a.w_next, a.param, cc, d, 1.f, w);
      load_param_chunk(a.b_next, a.param, cc, d, 0.f, b);
#pragma unroll
      for (int i = 0; i < kVec; ++i) p[c][i] = fmaf((h[c][i] - mean_h) * r_h, w[i], b[i]);
      store_chunk<T>(static_cast<S*>(a.n) + base, cc, d, p[c]);
    }
  }
  if (a.stats != nullptr && threadIdx.x % TPR == 0) {
    const float st[4] = {mean_y, r_y, mean_h, r_h};
    __builtin_memcpy(a.stats + row * 4, st, sizeof(st));
  }
}

struct NormGradArgs {
  const void *h, *y, *w, *b, *gate, *scale, *w_next, *dh, *dn;
  const float* stats;
  void *dx, *dy, *dgate;
  float* partial;  // [sums][gridDim.x][d], then [gridDim.x] for a single scale
  int64_t T, d;
  int32_t param, gate_cols, scale_cols;
  int32_t slot_w, slot_b, slot_s, slot_wn, slot_bn;  // which sum, -1: not needed
  int32_t sums;
};

constexpr int kSums = 5;

// Backward of a row, and the sums over the rows: a thread owns the same
// columns of every row that its workgroup takes and keeps their sums in
// registers; the workgroup's rows are added through LDS at the end and the
// workgroups' sums by reduce_kernel, always in the same order.
template <typename TX, typename T, int TPR, int CH, bool LAYER>
__global__ void __launch_bounds__(norm_threads(TPR))
block_norm_backward_kernel(NormGradArgs a) {
  typedef typename elem<TX>::storage SX;
  typedef typename elem<T>::storage S;
  constexpr int kThreads = norm_threads(TPR);
  constexpr int kRows = kThreads / TPR;
  constexpr int kWaves = kThreads / kWave;
  __shared__ float s_red[2 * 3 * kWaves];
  __shared__ float s_fold[kRows > 1 ? kThreads * CH * kVec : 1];
  const int64_t d = a.d, c0 = (int64_t)(threadIdx.x % TPR) * kVec;
  const int sub = threadIdx.x / TPR;
  float acc[kSums][CH][kVec];
#pragma unroll
  for (int q = 0; q < kSums; ++q)
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < kVec; ++i) acc[q][c][i] = 0.f;
  float w[CH][kVec], wn[CH][kVec], sc[CH][kVec];
  const float s_all = a.scale != nullptr && a.scale_cols == 1 ? load_param(a.scale, a.param, 0) : 1.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t cc = c0 + c * TPR * kVec;
    load_param_chunk(a.w, a.param, cc, d, 1.f, w[c]);
    load_param_chunk(a.w_next, a.param, cc, d, 1.f, wn[c]);
    load_param_chunk(a.scale_cols == 1 ? nullptr : a.scale, a.param, cc, d, s_all, sc[c]);
  }
  const float inv_d = 1.f / (float)d;
  RowSum<TPR, 3> sum3{s_red};
  const int64_t step = (int64_t)gridDim.x * kRows;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.T; r0 += step) {
    const int64_t row = r0 + sub;
    const bool live = row < a.T;  // only rows narrower than a wave's can be dead
    const int64_t base = (live ? row : 0) * d;
    float st[4];
    __builtin_memcpy(st, a.stats + (live ? row : 0) * 4, sizeof(st));
    float D[CH][kVec], y[CH][kVec];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t cc = c0 + c * TPR * kVec;
      if (a.dh != nullptr) {
        load_chunk<TX>(static_cast<const SX*>(a.dh) + base, cc, d, D[c]);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) D[c][i] = 0.f;
      }
    }
    if (a.dn != nullptr) {
      float hh[CH][kVec], u[CH][kVec];
      float t[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int64_t cc = c0 + c * TPR * kVec;
        load_chunk<TX>(static_cast<const SX*>(a.h) + base, cc, d, hh[c]);
        load_chunk<T>(static_cast<const S*>(a.dn) + base, cc, d, u[c]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          hh[c][i] = cc + i < d ? (hh[c][i] - st[2]) * st[3] : 0.f;
          if (live) {
            acc[3][c][i] = fmaf(u[c][i], hh[c][i], acc[3][c][i]);
            if constexpr (LAYER) acc[4][c][i] += u[c][i];
          }
          u[c][i] *= wn[c][i];
          t[0] += u[c][i];
          t[1] = fmaf(u[c][i], hh[c][i], t[1]);
        }
      }
      sum3(t);
      const float m0 = LAYER ? t[0] * inv_d : 0.f, m1 = t[1] * inv_d;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          D[c][i] = fmaf(st[3], u[c][i] - m0 - hh[c][i] * m1, D[c][i]);
    }
    if (a.dx != nullptr && live) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        store_chunk<TX>(static_cast<SX*>(a.dx) + base, c0 + c * TPR * kVec, d, D[c]);
    }
    if (a.y == nullptr) continue;
    const float g_row = a.gate != nullptr && a.gate_cols == 1
                            ? elem<T>::load(static_cast<const S*>(a.gate)[live ? row : 0]) : 1.f;
    float t[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t cc = c0 + c * TPR * kVec;
      float b[kVec], g[kVec], dg[kVec];
      load_chunk<T>(static_cast<const S*>(a.y) + base, cc, d, y[c]);
      load_param_chunk(a.b, a.param, cc, d, 0.f, b);
      if (a.gate != nullptr && a.gate_cols != 1) {
        load_chunk<T>(static_cast<const S*>(a.gate) + base, cc, d, g);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) g[i] = g_row;
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        y[c][i] = cc + i < d ? (y[c][i] - st[0]) * st[1] : 0.f;
        const float p = fmaf(y[c][i], w[c][i], b[i]);
        const float Dv = cc + i < d ? D[c][i] : 0.f;
        const float dgp = Dv * p;
        dg[i] = dgp * sc[c][i];
        t[2] += dg[i];
        const float dp = Dv * sc[c][i] * g[i];
        if (live) {
          acc[0][c][i] = fmaf(dp, y[c][i], acc[0][c][i]);
          if constexpr (LAYER) acc[1][c][i] += dp;
          acc[2][c][i] = fmaf(dgp, g[i], acc[2][c][i]);
        }
        D[c][i] = dp * w[c][i];
        t[0] += D[c][i];
        t[1] = fmaf(D[c][i], y[c][i], t[1]);
      }
      if (a.dgate != nullptr && a.gate_cols != 1 && live)
        store_chunk<T>(static_cast<S*>(a.dgate) + base, cc, d, dg);
    }
    sum3(t);
    if (a.dgate != nullptr && a.gate_cols == 1 && live && threadIdx.x % TPR == 0)
      static_cast<S*>(a.dgate)[row] = elem<T>::store(t[2]);
    if (a.dy != nullptr && live) {
      // without a norm's weight p = y: nothing to project out
      const float m0 = LAYER && a.w != nullptr ? t[0] * inv_d : 0.f;
      const float m1 = a.w != nullptr ? t[1] * inv_d : 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) y[c][i] = st[1] * (D[c][i] - m0 - y[c][i] * m1);
        store_chunk<T>(static_cast<S*>(a.dy) + base, c0 + c * TPR * kVec, d, y[c]);
      }
    }
  }
  if (a.sums == 0 && a.slot_s < 0) return;
  const int slots[kSums] = {a.slot_w, a.slot_b, a.slot_s, a.slot_wn, a.slot_bn};
#pragma unroll
  for (int q = 0; q < kSums; ++q) {
    if (slots[q] < 0) continue;
    if constexpr (kRows > 1) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < kVec; ++i) s_fold[(c * kVec + i) * kThreads + threadIdx.x] = acc[q][c][i];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            float s = 0.f;
            for (int r = 0; r < kRows; ++r) s += s_fold[(c * kVec + i) * kThreads + r * TPR + threadIdx.x];
            acc[q][c][i] = s;
          }
      }
    }
    if (q == 2 && a.scale_cols == 1) {
      float t[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < kVec; ++i) t[0] += acc[q][c][i];
      sum3(t);
      if (threadIdx.x == 0) a.partial[(int64_t)a.sums * gridDim.x * d + blockIdx.x] = t[0];
    } else if (sub == 0) {
      float* out = a.partial + ((int64_t)slots[q] * gridDim.x + blockIdx.x) * d;
#pragma unroll
      for (int c = 0; c < CH; ++c) store_chunk<float>(out, c0 + c * TPR * kVec, d, acc[q][c]);
    }
  }
}

struct ReduceArgs {
  const float* partial;
  int64_t d;
  int32_t blocks, param, sums;
  void* out[kSums];  // by slot
  void* scale;       // the single scale's gradient, or null
};

// The parameters' gradients: 64 columns per workgroup, its four waves take
// every fourth partial sum, in a fixed order. blockIdx.y past the sums: the
// single scale.
__global__ void __launch_bounds__(256) norm_reduce_kernel(ReduceArgs a) {
  __shared__ float s_sum[4][kWave];
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  if ((int)blockIdx.y == a.sums) {
    if (blockIdx.x != 0 || wave != 0) return;
    const float* p = a.partial + (int64_t)a.sums * a.blocks * a.d;
    float sum = 0.f;
    for (int i = lane; i < a.blocks; i += kWave) sum += p[i];
    sum = wave_sum(sum);
    if (lane == 0) store_param(a.scale, a.param, 0, sum);
    return;
  }
  const int64_t i = (int64_t)blockIdx.x * kWave + lane;
  const float* p = a.partial + (int64_t)blockIdx.y * a.blocks * a.d;
  float sum = 0.f;
  if (i < a.d) {
#pragma unroll 8
    for (int b = wave; b < a.blocks; b += 4) sum += p[(int64_t)b * a.d + i];
  }
  s_sum[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && i < a.d)
    store_param(a.out[blockIdx.y], a.param, i,
                (s_sum[0][lane] + s_sum[1][lane]) + (s_sum[2][lane] + s_sum[3][lane]));
}

// f(threads of a row, its chunks a thread) for a width. A row takes the
// fewest threads that hold it eight columns each; the set is coarse (16, 64,
// then powers of two) to keep the instantiations few.
template <typename F>
void by_width(int64_t d, F&& f) {
  const auto one = std::integral_constant<int, 1>();
  if (d <= 16 * kVec) f(std::integral_constant<int, 16>(), one);
  else if (d <= 64 * kVec) f(std::integral_constant<int, 64>(), one);
  else if (d <= 128 * kVec) f(std::integral_constant<int, 128>(), one);
  else if (d <= 256 * kVec) f(std::integral_constant<int, 256>(), one);
  else if (d <= 512 * kVec) f(std::integral_constant<int, 512>(), one);
  else if (d <= 1024 * kVec) f(std::integral_constant<int, 1024>(), one);
  else f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
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

int row_threads(int64_t d) {
  int t = 0;
  by_width(d, [&](auto tpr, auto) { t = decltype(tpr)::value; });
  return t;
}

// Workgroups of the backward: by the sizes alone (the order of the
// parameters' sums is the same on every device).
int64_t backward_blocks(int64_t T, int64_t d) {
  const int tpr = row_threads(d);
  const int64_t rows = norm_threads(tpr) / tpr;
  const int64_t most = tpr <= 256 ? 1024 : tpr == 512 ? 512 : 256;
  return std::max<int64_t>(1, std::min(most, ceil_div(T, rows)));
}

int check_norm(int x_dtype, int dtype, int param, int kind, int64_t T, int64_t d) {
  if (by_types(x_dtype, dtype, [](auto, auto) { return (int)NT_OK; }) != NT_OK) return NT_ERR_DTYPE;
  if (param != NT_F32 && param != NT_F16 && param != NT_BF16) return NT_ERR_DTYPE;
  if ((kind != NT_NORM_RMS && kind != NT_NORM_LAYER) || T < 0 || d < 1) return NT_ERR_INVALID_ARG;
  if (d > kMaxNormWidth || T > INT32_MAX) return NT_ERR_TOO_LARGE;
  return NT_OK;
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int nt_block_norm(int x_dtype, int dtype, int param_dtype, int kind, const void* x, const void* y,
                  const void* w, const void* b, const void* gate, int64_t gate_cols,
                  const void* scale, int64_t scale_cols, const void* w_next, const void* b_next,
                  float eps, int64_t T, int64_t d, void* h, void* n, float* stats,
                  hipStream_t stream) {
  const int st = check_norm(x_dtype, dtype, param_dtype, kind, T, d);
  if (st != NT_OK) return st;
  if (gate != nullptr && gate_cols != 1 && gate_cols != d) return NT_ERR_INVALID_ARG;
  if (scale != nullptr && scale_cols != 1 && scale_cols != d) return NT_ERR_INVALID_ARG;
  // a bias or gate has nothing to act on, or rms norms none at all
  if ((b != nullptr && (w == nullptr || kind == NT_NORM_RMS)) ||
      (b_next != nullptr && (w_next == nullptr || kind == NT_NORM_RMS)) ||
      (T > 0 && y == nullptr &&
       (w != nullptr || gate != nullptr || scale != nullptr || w_next == nullptr)))
    return NT_ERR_INVALID_ARG;
  if (T == 0) return NT_OK;  // tensors of no tokens may have no address
  if (x == nullptr || (y != nullptr && h == nullptr) || (w_next != nullptr && n == nullptr))
    return NT_ERR_INVALID_ARG;
  const NormArgs a = {x, y, w, b, gate, scale, w_next, b_next, h, n, stats, T, d, eps, param_dtype,
                      (int32_t)gate_cols, (int32_t)scale_cols};
  return by_types(x_dtype, dtype, [&](auto tx, auto t) {
    by_width(d, [&](auto tpr, auto ch) {
      constexpr int TPR = decltype(tpr)::value, CH = decltype(ch)::value;
      constexpr int threads = norm_threads(TPR);
      const dim3 grid((unsigned)ceil_div(T, (int64_t)(threads / TPR)));
      if (kind == NT_NORM_LAYER)
        hipLaunchKernelGGL((block_norm_kernel<decltype(tx), decltype(t), TPR, CH, true>), grid,
                           dim3(threads), 0, stream, a);
      else
        hipLaunchKernelGGL((block_norm_kernel<decltype(tx), decltype(t), TPR, CH, false>), grid,
                           dim3(threads), 0, stream, a);
    });
    return launch_status();
  });
}

size_t nt_block_norm_backward_workspace_bytes(int64_t T, int64_t d) {
  if (T < 0 || d < 1 || d > kMaxNormWidth || T > INT32_MAX) return 0;
  return (size_t)backward_blocks(T, d) * (size_t)(kSums * d + 1) * 4;
}

int nt_block_norm_backward(int x_dtype, int dtype, int param_dtype, int kind, const void* h,
                           const void* y, const void* w, const void* b, const void* gate,
                           int64_t gate_cols, const void* scale, int64_t scale_cols,
                           const void* w_next, const float* stats, const void* dh, const void* dn,
                           int64_t T, int64_t d, void* dx, void* dy, void* dgate, void* dscale,
                           void* dw, void* db, void* dw_next, void* db_next, void* ws,
                           size_t ws_bytes, hipStream_t stream) {
  const int st = check_norm(x_dtype, dtype, param_dtype, kind, T, d);
  if (st != NT_OK) return st;
  if (gate != nullptr && gate_cols != 1 && gate_cols != d) return NT_ERR_INVALID_ARG;
  if (scale != nullptr && scale_cols != 1 && scale_cols != d) return NT_ERR_INVALID_ARG;
  if ((T > 0 && y == nullptr &&
       (w != nullptr || gate != nullptr || scale != nullptr || dy != nullptr)) ||
      (T > 0 && dgate != nullptr && gate == nullptr) || (dn != nullptr && w_next == nullptr) ||
      (dscale != nullptr && scale == nullptr) || (dw != nullptr && w == nullptr) ||
      (dw_next != nullptr && w_next == nullptr) || (db != nullptr && w == nullptr) ||
      (db_next != nullptr && w_next == nullptr) ||
      (kind == NT_NORM_RMS && (b != nullptr || db != nullptr || db_next != nullptr)))
    return NT_ERR_INVALID_ARG;
  // a sum each; a scale of one value has its own place behind them
  void* const outs[kSums] = {dw, db, scale_cols == 1 ? nullptr : dscale, dw_next, db_next};
  const bool one = dscale != nullptr && scale_cols == 1;
  ReduceArgs r = {};
  int32_t slot[kSums], sums = 0;
  for (int q = 0; q < kSums; ++q) {
    slot[q] = outs[q] != nullptr ? sums : -1;
    if (outs[q] != nullptr) r.out[sums++] = outs[q];
  }
  const bool reduce = sums > 0 || one;
  const int64_t blocks = backward_blocks(T, d);
  const size_t need = (size_t)blocks * (size_t)(sums * d + one) * 4;
  if (T > 0 && (h == nullptr || stats == nullptr)) return NT_ERR_INVALID_ARG;
  if (reduce && (ws == nullptr || ws_bytes < need)) return NT_ERR_WORKSPACE;
  const NormGradArgs a = {h, y, w, b, gate, scale, w_next, dh, dn, stats, dx, dy, dgate,
                          static_cast<float*>(ws), T, d, param_dtype, (int32_t)gate_cols,
                          (int32_t)scale_cols, slot[0], slot[1], one ? 0 : slot[2], slot[3],
                          slot[4], sums};
  // no tokens: one workgroup writes the sums' zeros
  if (T == 0 && !reduce) return NT_OK;
  const int rc = by_types(x_dtype, dtype, [&](auto tx, auto t) {
    by_width(d, [&](auto tpr, auto ch) {
      constexpr int TPR = decltype(tpr)::value, CH = decltype(ch)::value;
      constexpr int threads = norm_threads(TPR);
      if (kind == NT_NORM_LAYER)
        hipLaunchKernelGGL((block_norm_backward_kernel<decltype(tx), decltype(t), TPR, CH, true>),
                           dim3((unsigned)blocks), dim3(threads), 0, stream, a);
      else
        hipLaunchKernelGGL((block_norm_backward_kernel<decltype(tx), decltype(t), TPR, CH, false>),
                           dim3((unsigned)blocks), dim3(threads), 0, stream, a);
    });
    return launch_status();
  });
  if (rc != NT_OK || !reduce) return rc;
  r.partial = static_cast<const float*>(ws);
  r.d = d;
  r.blocks = (int32_t)blocks;
  r.param = param_dtype;
  r.sums = sums;
  r.scale = one ? dscale : nullptr;
  hipLaunchKernelGGL(norm_reduce_kernel,
                     dim3((unsigned)ceil_div(d, (int64_t)kWave), (unsigned)(sums + one)), dim3(256),
                     0, stream, r);
  return launch_status();
}

}  // extern "C"
