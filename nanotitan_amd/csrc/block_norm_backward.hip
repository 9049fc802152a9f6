// Gradients of the block norms (block_norm.hip). With D = dh + dN(dn; h, w') and
// dN(d) = r (u - [mean u] - vhat mean(u vhat)) for u = d w, vhat = (v - m) r, [.]
// for layer norms:
//   dx = D,  dp = D s g,  dy = dN(dp; y, w),  dg = D s p,  ds = sum_t D g p,
//   dw = sum_t dp yhat,  db = sum_t dp,  dw' = sum_t dn hhat,  db' = sum_t dn.
//
// Bound by HBM, as the forward. A thread owns the same columns of every row
// that its workgroup takes and keeps the parameters' sums over them in
// registers; the workgroup's rows are added through LDS at the end and the
// workgroups' sums by a second launch, always in the same order. Four waves a
// SIMD have to fit (128 registers): the parameters are parked in LDS (layer
// norms of 131,072 x 512: 222 -> 160 us, of 16,384 x 4,096: 307 -> 199).
//
// Measured on MI355X (a copy: 5.65 TB/s), bf16: 16,384 x 4,096 rms 160 us
// (5.0 TB/s), layer 172 (4.7); 131,072 x 512 156 and 161 (5.2, 5.0); the sums'
// launch is 5 to 8 us of each. Above 8,192 columns a thread holds sixteen and
// the sums no longer fit its registers: 4,096 x 16,384 rms 215 (3.7), layer 424
// (1.9).
#include "block_norm.hpp"

namespace nt {
namespace {

using namespace norm;

// Sums over the tokens, a column each. The scale and the weight are the same
// for every token, so that two serve the branch's three gradients:
//   A = sum D g yhat,  B = sum D g:  dw = s A,  db = s B,  ds = w A + b B.
enum { kSumA = 0, kSumB = 1, kSumNext = 2, kSumNextBias = 3, kSums = 4 };

struct NormGradArgs {
  const void *h, *y, *w, *b, *gate, *scale, *w_next, *dh, *dn;
  const float* stats;
  void *dx, *dy, *dgate;
  float* partial;  // [sums][gridDim.x][d], then [gridDim.x] for a single scale
  int64_t T;
  int32_t d, param, gate_cols, scale_cols;
  int32_t slot[kSums];  // which of the sums, -1: not needed
  int32_t sums;
  bool one;  // the single scale's gradient is wanted
};

// The parameters of a thread's columns, where only it reads them: a row needs
// them twice for a moment, and the registers go to the sums.
template <int SETS, int CH, int V, int THREADS>
struct Parked {
  static constexpr int W = V % 4 == 0 ? 4 : 1;  // values side by side
  typedef float F __attribute__((ext_vector_type(W)));
  static constexpr int kSize = SETS * CH * V / W * THREADS;
  F* s;
  __device__ __forceinline__ F* at(int set, int k) const {
    return s + (set * CH + k) * (V / W) * THREADS + threadIdx.x;
  }
  __device__ __forceinline__ void put(int set, int k, const float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; i += W) __builtin_memcpy(at(set, k) + i / W * THREADS, v + i, sizeof(F));
  }
  __device__ __forceinline__ void get(int set, int k, float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; i += W) __builtin_memcpy(v + i, at(set, k) + i / W * THREADS, sizeof(F));
  }
};

template <typename TX, typename T, typename SH, bool LAYER, int MODE>
__global__ void __launch_bounds__(block_threads(SH::TPR))
__attribute__((amdgpu_waves_per_eu(LAYER || SH::TPR >= 512 ? 4 : 1)))
block_norm_backward_kernel(NormGradArgs a) {
  typedef typename elem<T>::storage S;
  constexpr int V = SH::V, TPR = SH::TPR, CH = SH::CH;
  constexpr int kThreads = block_threads(TPR), kRows = kThreads / TPR;
  __shared__ float s_red[RowSum<TPR, 3>::kSize];
  __shared__ float s_fold[kRows > 1 ? kThreads * CH * V : 1];
  RowSum<TPR, 3> sum{s_red};
  enum { kSW, kNext, kSB };
  constexpr bool kParkSB = LAYER && CH == 1;  // three sets of 16,384 exceed the LDS
  typedef Parked<kParkSB ? 3 : 2, CH, V, kThreads> Params;
  __shared__ typename Params::F s_params[Params::kSize];
  const Params params{s_params};
  // a wave's rows are one: its addresses stay scalar
  const int sub =
      TPR >= kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x / TPR) : threadIdx.x / TPR;
  Chunk<V> c[CH];
  float acc[kSums][CH][V], sb[CH][V];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    c[k] = Chunk<V>((k * TPR + threadIdx.x % TPR) * V, a.d);
    float sw[V], wn[V];
    if constexpr (MODE != kPre) {
      load_scaled<V, LAYER>(a.w, a.b, a.scale, a.scale_cols, a.param, c[k], sw, sb[k]);
      params.put(kSW, k, sw);
      if constexpr (kParkSB) params.put(kSB, k, sb[k]);
    }
    load_params<V>(a.w_next, a.param, c[k], 1.f, wn);
    params.put(kNext, k, wn);
#pragma unroll
    for (int q = 0; q < kSums; ++q)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[q][k][i] = 0.f;
  }
  const float inv_d = 1.f / (float)a.d;
  // a missing gradient's loads go to h, and count for nothing
  const bool has_dh = a.dh != nullptr, has_dn = a.dn != nullptr;
  const void *const dh = has_dh ? a.dh : a.h, *const dn = has_dn ? a.dn : a.h;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + sub;
  Raw<TX, V> rd[CH], rh[CH];
  Raw<T, V> rn[CH], ry[CH], rg[CH];
  float st[4];
  auto load = [&](int64_t r) {
    const int64_t at = r < a.T ? r : a.T - 1, base = at * a.d;
    __builtin_memcpy(st, a.stats + at * 4, sizeof(st));
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      rd[k] = load_raw<TX, V>(dh, base, c[k]);
      rh[k] = load_raw<TX, V>(a.h, base, c[k]);
      rn[k] = load_raw<T, V>(dn, base, c[k]);
      if constexpr (MODE != kPre) ry[k] = load_raw<T, V>(a.y, base, c[k]);
      if constexpr (MODE == kGated) rg[k] = load_raw<T, V>(a.gate, base, c[k]);
    }
  };
  for (int64_t first = (int64_t)blockIdx.x * kRows; first < a.T; first += step, row += step) {
    const bool live = row < a.T;  // rows that share a workgroup may be past the end
    const int64_t base = row * a.d;
    asm volatile("" ::: "memory");  // the parameters stay parked
    load(row);
    const float mean_y = st[0], r_y = st[1], mean_h = st[2], r_h = st[3];
    // Columns that a chunk does not own count in the row's sums with parameters
    // of zero, and their own sums are not stored.
    float D[CH][V], hh[CH][V], u[CH][V], y[CH][V], g[CH][V];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      all_values<TX, V>(rd[k], D[k]);
      all_values<TX, V>(rh[k], hh[k]);
      all_values<T, V>(rn[k], u[k]);
      if constexpr (MODE != kPre) all_values<T, V>(ry[k], y[k]);
      if constexpr (MODE == kGated) all_values<T, V>(rg[k], g[k]);
    }
    if (!has_dh) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) D[k][i] = 0.f;
    }
    if (has_dn) {
      float t[LAYER ? 2 : 1] = {};
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        float wn[V];
        params.get(kNext, k, wn);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          hh[k][i] = (hh[k][i] - mean_h) * r_h;
          if (live) {
            acc[kSumNext][k][i] = fmaf(u[k][i], hh[k][i], acc[kSumNext][k][i]);
            if constexpr (LAYER) acc[kSumNextBias][k][i] += u[k][i];
          }
          u[k][i] *= wn[i];
          t[0] = fmaf(u[k][i], hh[k][i], t[0]);
          if constexpr (LAYER) t[1] += u[k][i];
        }
      }
      sum(t);
      float m0 = 0.f, m1 = t[0] * inv_d;
      if constexpr (LAYER) m0 = t[1] * inv_d;
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
          D[k][i] = fmaf(r_h, u[k][i] - m0 - hh[k][i] * m1, D[k][i]);
    }
    if (a.dx != nullptr && live) {
#pragma unroll
      for (int k = 0; k < CH; ++k) store_chunk<TX, V>(a.dx, base, c[k], D[k]);
    }
    if constexpr (MODE != kPre) {
      float g_row = 1.f;
      if (MODE == kPost && a.gate != nullptr)
        g_row = elem<T>::load(static_cast<const S*>(a.gate)[live ? row : a.T - 1]);
      constexpr int kGate = LAYER ? 2 : 1;  // a row's gate: its sum is the last
      float t[kGate + (MODE == kPost)] = {};
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        float dg[V], sw[V];
        params.get(kSW, k, sw);
        if constexpr (kParkSB) params.get(kSB, k, sb[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float gi = MODE == kGated ? g[k][i] : g_row;
          const float Dv = D[k][i];
          y[k][i] = (y[k][i] - mean_y) * r_y;
          // s g p's derivative by g, and D g: times s w it is u of dN, summed A and B
          dg[i] = Dv * (LAYER ? fmaf(y[k][i], sw[i], sb[k][i]) : y[k][i] * sw[i]);
          if constexpr (MODE == kPost) t[kGate] += dg[i];
          const float Dg = Dv * gi;
          if (live) {
            acc[kSumA][k][i] = fmaf(Dg, y[k][i], acc[kSumA][k][i]);
            if constexpr (LAYER) acc[kSumB][k][i] += Dg;
          }
          D[k][i] = Dg * sw[i];
          t[0] = fmaf(D[k][i], y[k][i], t[0]);
          if constexpr (LAYER) t[1] += D[k][i];
        }
        if (MODE == kGated && a.dgate != nullptr && live)
          store_chunk<T, V>(a.dgate, base, c[k], dg);
      }
      sum(t);
      if constexpr (MODE == kPost)
        if (a.dgate != nullptr && live && threadIdx.x % TPR == 0)
          static_cast<S*>(a.dgate)[row] = elem<T>::store(t[kGate]);
      if (a.dy != nullptr && live) {
        // without a norm's weight p = y: nothing to project out, and whatever y
        // holds (an infinity times zero would be a NaN) dy is D
        const bool norm = a.w != nullptr;
        float m0 = 0.f, m1 = t[0] * inv_d;
        if constexpr (LAYER) m0 = t[1] * inv_d;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            y[k][i] = norm ? r_y * (D[k][i] - m0 - y[k][i] * m1) : D[k][i];
          store_chunk<T, V>(a.dy, base, c[k], y[k]);
        }
      }
    }
  }
#pragma unroll
  for (int q = 0; q < kSums; ++q) {
    if (a.slot[q] < 0) continue;
    if constexpr (kRows > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s_fold[(k * V + i) * kThreads + threadIdx.x] = acc[q][k][i];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int k = 0; k < CH; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
              s += s_fold[(k * V + i) * kThreads + r * TPR + threadIdx.x];
            acc[q][k][i] = s;
          }
      }
    }
    if (sub == 0) {
      const int64_t base = ((int64_t)a.slot[q] * gridDim.x + blockIdx.x) * a.d;
#pragma unroll
      for (int k = 0; k < CH; ++k) store_chunk<float, V>(a.partial, base, c[k], acc[q][k]);
    }
  }
  if (MODE != kPre && a.one) {
    float t[1] = {0.f};
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float w[V], b[V];
      load_params<V>(a.w, a.param, c[k], 1.f, w);
      load_params<V>(a.b, a.param, c[k], 0.f, b);
#pragma unroll
      for (int i = 0; i < V; ++i)
        t[0] += w[i] * acc[kSumA][k][i] + (LAYER ? b[i] * acc[kSumB][k][i] : 0.f);
    }
    sum(t);
    if (threadIdx.x == 0) a.partial[(int64_t)a.sums * gridDim.x * a.d + blockIdx.x] = t[0];
  }
}

struct ReduceArgs {
  const float* partial;
  const void *w, *b, *scale;
  int64_t d;
  int32_t blocks, param, scale_cols, sums, jobs;
  struct Job {
    void* out;
    int32_t first, second;  // the sums that it takes (slots; -1: none)
    bool scaled, weighted;  // the first times the scale, or times w
  } job[5];
  void* one;  // the single scale's gradient, or null
};

// The parameters' gradients: 16 columns per workgroup, 16 groups of 16 lanes
// taking every sixteenth partial sum, in a fixed order. blockIdx.y past the
// jobs: the single scale.
constexpr int kReduceCols = 16;
__global__ void __launch_bounds__(256) norm_reduce_kernel(ReduceArgs a) {
  constexpr int kGroups = 256 / kReduceCols;
  __shared__ float s_sum[2][kGroups][kReduceCols];
  if ((int)blockIdx.y == a.jobs) {
    if (blockIdx.x != 0 || threadIdx.x >= kWave) return;
    const float* p = a.partial + (int64_t)a.sums * a.blocks * a.d;
    float sum = 0.f;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.blocks; i += kWave) sum += p[i];
    sum = wave_sum(sum);
    if (threadIdx.x == 0) store_param(a.one, a.param, 0, sum);
    return;
  }
  const ReduceArgs::Job job = a.job[blockIdx.y];
  const int col = threadIdx.x % kReduceCols, group = threadIdx.x / kReduceCols;
  const int64_t i = (int64_t)blockIdx.x * kReduceCols + col, at = i < a.d ? i : a.d - 1;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int slot = h == 0 ? job.first : job.second;
    float sum = 0.f;
    if (slot >= 0) {
      const float* p = a.partial + (int64_t)slot * a.blocks * a.d + at;
#pragma unroll 16
      for (int b = group; b < a.blocks; b += kGroups) sum += p[(int64_t)b * a.d];
    }
    s_sum[h][group][col] = sum;
  }
  __syncthreads();
  if (group == 0 && i < a.d) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < kGroups; ++g) sum[h] += s_sum[h][g][col];
    float v = sum[0];
    if (job.scaled && a.scale != nullptr)
      v *= load_param(a.scale, a.param, a.scale_cols == 1 ? 0 : i);
    if (job.weighted && a.w != nullptr) v *= load_param(a.w, a.param, i);
    if (job.second >= 0) v += sum[1] * load_param(a.b, a.param, i);
    store_param(job.out, a.param, i, v);
  }
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

size_t nt_block_norm_backward_workspace_bytes(int64_t T, int64_t d) {
  if (T < 0 || d < 1 || d > norm::kMaxWidth || T > INT32_MAX) return 0;
  return (size_t)norm::blocks_of(T, d, 4) * (size_t)(kSums * d + 1) * 4;
}

int nt_block_norm_backward(int x_dtype, int dtype, int param_dtype, int kind, const void* h,
                           const void* y, const void* w, const void* b, const void* gate,
                           int64_t gate_cols, const void* scale, int64_t scale_cols,
                           const void* w_next, const float* stats, const void* dh, const void* dn,
                           int64_t T, int64_t d, void* dx, void* dy, void* dgate, void* dscale,
                           void* dw, void* db, void* dw_next, void* db_next, void* ws,
                           size_t ws_bytes, hipStream_t stream) {
  const int st = norm::check_norm(x_dtype, dtype, param_dtype, kind, T, d);
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
  const bool one = dscale != nullptr && scale_cols == 1, channel = dscale != nullptr && !one;
  const int64_t blocks = norm::blocks_of(T, d, 4);
  NormGradArgs a = {h, y, w, b, gate, scale, w_next, dh, dn, stats, dx, dy, dgate,
                    static_cast<float*>(ws), T, (int32_t)d, param_dtype, (int32_t)gate_cols,
                    (int32_t)scale_cols, {-1, -1, -1, -1}, 0, one};
  if (dw != nullptr || dscale != nullptr) a.slot[kSumA] = a.sums++;
  if (db != nullptr || (dscale != nullptr && b != nullptr)) a.slot[kSumB] = a.sums++;
  if (dw_next != nullptr) a.slot[kSumNext] = a.sums++;
  if (db_next != nullptr) a.slot[kSumNextBias] = a.sums++;
  if (T > 0 && (h == nullptr || stats == nullptr)) return NT_ERR_INVALID_ARG;
  if (a.sums > 0 && (ws == nullptr || ws_bytes < (size_t)blocks * (size_t)(a.sums * d + one) * 4))
    return NT_ERR_WORKSPACE;
  if (T == 0 && a.sums == 0) return NT_OK;  // else one workgroup writes the sums' zeros
  const int rc = norm::by_types(x_dtype, dtype, [&](auto tx, auto t) {
    norm::by_width(d, [&](auto shape) {
      const bool gate_each = gate != nullptr && gate_cols == d && d > 1;
      norm::by_mode(y != nullptr || T == 0, gate_each, [&](auto mode) {
        typedef decltype(shape) SH;
        constexpr int M = decltype(mode)::value;
        const dim3 grid((unsigned)blocks), block(norm::block_threads(SH::TPR));
        if (kind == NT_NORM_LAYER)
          hipLaunchKernelGGL((block_norm_backward_kernel<decltype(tx), decltype(t), SH, true, M>),
                             grid, block, 0, stream, a);
        else
          hipLaunchKernelGGL((block_norm_backward_kernel<decltype(tx), decltype(t), SH, false, M>),
                             grid, block, 0, stream, a);
      });
    });
    return launch_status();
  });
  if (rc != NT_OK || a.sums == 0) return rc;
  ReduceArgs r = {static_cast<const float*>(ws), w, b, scale, d, (int32_t)blocks, param_dtype,
                  (int32_t)scale_cols, a.sums, 0, {}, one ? dscale : nullptr};
  if (dw != nullptr) r.job[r.jobs++] = {dw, a.slot[kSumA], -1, true, false};
  if (db != nullptr) r.job[r.jobs++] = {db, a.slot[kSumB], -1, true, false};
  if (channel)
    r.job[r.jobs++] = {dscale, a.slot[kSumA], b != nullptr ? a.slot[kSumB] : -1, false, true};
  if (dw_next != nullptr) r.job[r.jobs++] = {dw_next, a.slot[kSumNext], -1, false, false};
  if (db_next != nullptr) r.job[r.jobs++] = {db_next, a.slot[kSumNextBias], -1, false, false};
  hipLaunchKernelGGL(norm_reduce_kernel,
                     dim3((unsigned)ceil_div(d, (int64_t)kReduceCols), (unsigned)(r.jobs + one)),
                     dim3(256), 0, stream, r);
  return launch_status();
}

}  // extern "C"
