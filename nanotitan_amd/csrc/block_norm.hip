// Norms before and after a block, fused with the block's gate and residual
// scale.
//
//   N(v) = (v - m) r w + b   rms:   m = 0,       r = 1 / sqrt(mean v^2 + eps)
//                            layer: m = mean v,  r = 1 / sqrt(mean (v - m)^2 + eps)
//   p = N(y; w, b)  (p = y without a weight),  h = x + s g p rounded to x's
//   type,  n = N(h; w', b') of h as it is held.
//
// Bound by HBM: one pass over each row, its values held in registers between
// the sums over the row and their use, the parameters read once per workgroup.
// The loads of a row go out together; the other waves of a SIMD hide them
// (with the next row's loads kept in flight instead, fewer waves fit: 122
// against 112 us at 16,384 x 4,096). A layer norm's workgroup that has its CU
// alone keeps the next row in flight (8,192 x 8,192, bf16: 124 -> 104 us), but
// not where a thread's rows fill the registers (16,384 columns).
//
// At 40 instructions a value, 16-bit rows would wait for the vector units: so
// columns that a thread does not own are cleared two at a time and once, sums
// go by lane moves, and the root is one instruction.
//
// Measured on MI355X (a copy: 5.65 TB/s), bf16, norm, residual and next norm:
// 16,384 x 4,096 rms 101 us (5.3 TB/s), layer 105 (5.1); 131,072 x 512 108 and
// 104 (5.0, 5.1); with an elementwise gate 130 and 126 (5.2, 5.3).
#include "block_norm.hpp"

namespace nt {
namespace {

using namespace norm;

struct NormArgs {
  const void *x, *y, *w, *b, *gate, *scale, *w_next, *b_next;
  void *h, *n;
  float* stats;  // [T][4]: mean and r of y, mean and r of h (may be null)
  int64_t T;
  int32_t d;
  float eps;
  int32_t param, gate_cols, scale_cols;
};

// mean and r of a row held in v (zeros where a chunk does not own a column).
template <typename SH, bool LAYER>
__device__ __forceinline__ void row_stats(const float (&v)[SH::CH][SH::V],
                                          const Chunk<SH::V> (&c)[SH::CH], float inv_d, float eps,
                                          RowSum<SH::TPR, 1>& sum, float& mean, float& r) {
  mean = 0.f;
  if constexpr (LAYER) {
    float t[1] = {0.f};
#pragma unroll
    for (int k = 0; k < SH::CH; ++k)
#pragma unroll
      for (int i = 0; i < SH::V; ++i) t[0] += v[k][i];
    sum(t);
    mean = t[0] * inv_d;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int k = 0; k < SH::CH; ++k)
#pragma unroll
    for (int i = 0; i < SH::V; ++i) {
      const float u = !LAYER || c[k].owns(i) ? v[k][i] - mean : 0.f;
      q[0] = fmaf(u, u, q[0]);
    }
  sum(q);
  // The instruction is within one unit in the last place, but for denormals,
  // which are scaled out of its way. (A root and a division in full were 40
  // instructions for each thread's eight values.)
  const float var = fmaf(q[0], inv_d, eps);
  const bool tiny = var < 0x1p-100f;
  r = __builtin_amdgcn_rsqf(tiny ? var * 0x1p+60f : var) * (tiny ? 0x1p+30f : 1.f);
}

template <typename TX, typename T, typename SH, bool LAYER, int MODE>
__global__ void __launch_bounds__(block_threads(SH::TPR)) block_norm_kernel(NormArgs a) {
  constexpr int V = SH::V, TPR = SH::TPR, CH = SH::CH;
  constexpr int kThreads = block_threads(TPR), kRows = kThreads / TPR;
  __shared__ float s_red[RowSum<TPR, 1>::kSize];
  RowSum<TPR, 1> sum{s_red};
  constexpr bool kAhead = LAYER && TPR >= 1024 && CH == 1;
  Chunk<V> c[CH];
  float sw[CH][V], sb[CH][V], wn[CH][V], bn[CH][V];  // s w, s b, w', b'
  const float inv_d = 1.f / (float)a.d;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    c[k] = Chunk<V>((k * TPR + threadIdx.x % TPR) * V, a.d);
    if constexpr (MODE != kPre)
      load_scaled<V, LAYER>(a.w, a.b, a.scale, a.scale_cols, a.param, c[k], sw[k], sb[k]);
    load_params<V>(a.w_next, a.param, c[k], 1.f, wn[k]);
    if constexpr (LAYER) load_params<V>(a.b_next, a.param, c[k], 0.f, bn[k]);
  }
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  Raw<TX, V> rx[CH];
  Raw<T, V> ry[CH], rg[CH];
  auto load = [&](int64_t r) {
    const int64_t base = (r < a.T ? r : a.T - 1) * a.d;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      rx[k] = load_raw<TX, V>(a.x, base, c[k]);
      if constexpr (MODE != kPre) ry[k] = load_raw<T, V>(a.y, base, c[k]);
      if constexpr (MODE == kGated) rg[k] = load_raw<T, V>(a.gate, base, c[k]);
    }
  };
  if constexpr (kAhead) load(row);
  for (int64_t first = (int64_t)blockIdx.x * kRows; first < a.T; first += step, row += step) {
    const bool live = row < a.T;  // rows that share a workgroup may be past the end
    const int64_t base = row * a.d;
    if constexpr (!kAhead) load(row);
    float h[CH][V], p[CH][V], g[CH][V];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      values<TX, V>(rx[k], c[k], h[k]);
      if constexpr (MODE != kPre) values<T, V>(ry[k], c[k], p[k]);
      // (a layer norm's row is NaN with any infinity in it, owned or not)
      if constexpr (MODE == kGated)
        all_values<T, V>(LAYER ? rg[k] : owned<T, V>(rg[k], c[k]), g[k]);
    }
    if constexpr (kAhead) load(row + step);
    // x, y and the parameters are zero where a chunk does not own a column, and so
    // is h, whose gate is cleared for it: an infinity times zero would be a NaN
    float mean_y = 0.f, r_y = 1.f, mean_h = 0.f, r_h = 1.f;
    if constexpr (MODE != kPre) {
      float g_row = 1.f;
      if (MODE == kPost && a.gate != nullptr)
        g_row = elem<T>::load(
            static_cast<const typename elem<T>::storage*>(a.gate)[live ? row : a.T - 1]);
      if (a.w != nullptr) row_stats<SH, LAYER>(p, c, inv_d, a.eps, sum, mean_y, r_y);
#pragma unroll
      for (int k = 0; k < CH; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float hat = (p[k][i] - mean_y) * r_y;
          const float v = LAYER ? fmaf(hat, sw[k][i], sb[k][i]) : hat * sw[k][i];
          h[k][i] = elem<TX>::load(
              to_bits<TX>(fmaf(MODE == kGated ? g[k][i] : g_row, v, h[k][i])));
        }
        if (live) store_chunk<TX, V>(a.h, base, c[k], h[k]);
      }
    }
    if (a.w_next != nullptr) {
      row_stats<SH, LAYER>(h, c, inv_d, a.eps, sum, mean_h, r_h);
#pragma unroll
      for (int k = 0; k < CH; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float hat = (h[k][i] - mean_h) * r_h;
          p[k][i] = LAYER ? fmaf(hat, wn[k][i], bn[k][i]) : hat * wn[k][i];
        }
        if (live) store_chunk<T, V>(a.n, base, c[k], p[k]);
      }
    }
    if (a.stats != nullptr && live && threadIdx.x % TPR == 0) {
      const float st[4] = {mean_y, r_y, mean_h, r_h};
      __builtin_memcpy(a.stats + row * 4, st, sizeof(st));
    }
  }
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
  const int st = norm::check_norm(x_dtype, dtype, param_dtype, kind, T, d);
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
  const NormArgs a = {x, y, w, b, gate, scale, w_next, b_next, h, n, stats, T, (int32_t)d, eps,
                      param_dtype, (int32_t)gate_cols, (int32_t)scale_cols};
  return norm::by_types(x_dtype, dtype, [&](auto tx, auto t) {
    norm::by_width(d, [&](auto shape) {
      norm::by_mode(y != nullptr, gate != nullptr && gate_cols == d && d > 1, [&](auto mode) {
        typedef decltype(shape) SH;
        constexpr int M = decltype(mode)::value;
        // Waves a SIMD. Of 6, workgroups of 16 waves would be one and a half a CU
        // (8,192 x 8,192, bf16, rms: 110 us, against 103); of 8, layer norms' sums
        // in turn are slower (16,384 x 4,096: 116 against 104).
        constexpr int kWaves = SH::TPR >= 1024 ? 8 : 6;
        const dim3 grid((unsigned)norm::blocks_of(T, d, kind == NT_NORM_LAYER ? 4 : kWaves));
        const dim3 block(norm::block_threads(SH::TPR));
        if (kind == NT_NORM_LAYER)
          hipLaunchKernelGGL((block_norm_kernel<decltype(tx), decltype(t), SH, true, M>), grid,
                             block, 0, stream, a);
        else
          hipLaunchKernelGGL((block_norm_kernel<decltype(tx), decltype(t), SH, false, M>), grid,
                             block, 0, stream, a);
      });
    });
    return launch_status();
  });
}

}  // extern "C"
