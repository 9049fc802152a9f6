// A whole MoE layer for the few tokens (at most 64) of a decode step:
//
//   l = x Wr^T (or given),  S_t = the k largest of l_t (ties to the lower id),
//   g = softmax of l over S_t,  out_t = sum_{e in S_t} g_te act(x_t W1_e) W2_e
//   with act(z) = silu(x W_gate) * (x W_val) or gelu(x W_up).
//
// With so few tokens the layer is one read of the chosen experts' weights:
// HBM bounds the large layers, latency and launches the small ones. So no row
// is packed: a workgroup finds an expert's tokens from 64-bit masks (bit t of
// expert e: token t chose e) and multiplies its tile of the weights with all of
// them at once on the matrix cores.
//
// Weights are [K, N] row-major and the matrix instruction wants each lane's
// eight k values of one column in a register quad. A lane loads eight rows of
// four neighbouring columns straight from memory and transposes them with byte
// permutes (one per two values): nothing but the tokens is read twice, nothing
// goes through LDS but the waves' partial sums at the end.
#include <algorithm>

#include "common.hpp"

namespace nt {
namespace {

constexpr int kMaxTokens = NT_FEW_TOKENS_MAX;
constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kCols = 64;   // columns of a tile: 16 lanes x 4
constexpr int kRowsMma = 16;
constexpr int kStep = 32;   // weight rows a wave takes at a time
constexpr int kSlots = 512;  // workgroups of the expert kernels: two on each of 256 CUs

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct FewArgs {
  const void* x;        // [T, d]
  const float* router;  // [E, d], or null
  const float* logits;  // [T, E], used without a router
  const void *w1, *w2;  // [E, d, f]; w2 null for gelu
  const void* w3;       // [E, f, d]
  int32_t T, E, k, splits;
  int64_t d, f;
  float* gates;    // [T, k]
  int32_t* topk;   // [T, k]
  void* out;       // [T, d]
  int32_t* inv;    // [T, k]: row of an assignment in hidden and partial
  void* hidden;    // [T k, f]
  float* partial;  // [splits][T k][d]
};

// ------------------------------------------------------------------ routing

// Choices in the order of nt_route_topk as one unsigned key, the larger first:
// the value's bits as an ordered integer (-0 as +0, every NaN below -inf), then
// the lower expert. 0: no choice.
__device__ __forceinline__ uint64_t choice_key(float z, int e) {
  const uint32_t u = __float_as_uint(z == 0.f ? 0.f : z);
  const uint32_t ordered = z != z ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
  return ((uint64_t)ordered << 32) | (uint32_t)~e;
}
__device__ __forceinline__ float choice_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u == 0u ? 0x7fc00000u : (u >> 31) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int choice_expert(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  const uint32_t lo = __shfl_xor((uint32_t)v, o, kWave);
  return ((uint64_t)__shfl_xor((uint32_t)(v >> 32), o, kWave) << 32) | lo;
}

// One token a workgroup: its logits (a wave takes every sixteenth expert, its
// lanes the columns), then the top-k by one wave.
constexpr int kRouteThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) few_route_kernel(FewArgs a) {
  typedef typename elem<T>::storage S;
  __shared__ float s_logit[NT_MAX_EXPERTS];
  const int t = blockIdx.x, lane = lane_id(), wave = threadIdx.x / kWave;
  if (a.router != nullptr) {
    const S* x = static_cast<const S*>(a.x) + (int64_t)t * a.d;
    for (int e = wave; e < a.E; e += kRouteThreads / kWave) {
      const float* w = a.router + (int64_t)e * a.d;
      float sum = 0.f;
      for (int64_t c = lane * 4; c < a.d; c += kWave * 4) {
        if (c + 4 <= a.d) {
          float wv[4];
          S xv[4];
          __builtin_memcpy(wv, w + c, sizeof(wv));
          __builtin_memcpy(xv, x + c, sizeof(xv));
#pragma unroll
          for (int i = 0; i < 4; ++i) sum = fmaf(elem<T>::load(xv[i]), wv[i], sum);
        } else {
          for (int64_t i = c; i < a.d; ++i) sum = fmaf(elem<T>::load(x[i]), w[i], sum);
        }
      }
      sum = wave_sum(sum);
      if (lane == 0) s_logit[e] = sum;
    }
  } else {
    for (int e = threadIdx.x; e < a.E; e += kRouteThreads) s_logit[e] = a.logits[(int64_t)t * a.E + e];
  }
  __syncthreads();
  if (wave != 0) return;
  // lane l holds experts l, l + 64, ...; the j-th choice stays with lane j
  constexpr int V = NT_MAX_EXPERTS / kWave;
  uint64_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * kWave + lane;
    key[v] = e < a.E ? choice_key(s_logit[e], e) : 0ull;
  }
  float value = -INFINITY, top = 0.f;
  int expert = 0;
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v)
      if (v * kWave < a.E) best = key[v] > best ? key[v] : best;
    for (int o = 1; o < kWave; o <<= 1) {
      const uint64_t other = shfl_xor64(best, o);
      best = other > best ? other : best;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * kWave < a.E) key[v] = key[v] == best ? 0ull : key[v];
    const float z = choice_value(best);
    if (j == 0) top = z;
    if (lane == j) {
      value = z;
      expert = choice_expert(best);
    }
  }
  const float p = lane < a.k ? expf(value - top) : 0.f;
  const float den = wave_sum(p);
  if (lane < a.k) {
    a.gates[t * a.k + lane] = p * (1.f / den);
    a.topk[t * a.k + lane] = expert;
  }
}

// ------------------------------------------------------------- expert tiles

// What every workgroup of the expert kernels finds out first: each expert's
// tokens, the first row of each (rows by expert, then token) and the experts
// that have any.
struct Plan {
  uint64_t mask[NT_MAX_EXPERTS];
  uint16_t first[NT_MAX_EXPERTS];
  uint16_t live[NT_MAX_EXPERTS];
  int32_t num_live;
};

__device__ __forceinline__ void make_plan(const FewArgs& a, Plan& s) {
  for (int e = threadIdx.x; e < a.E; e += kThreads) s.mask[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * a.k; i += kThreads)
    atomicOr(reinterpret_cast<unsigned long long*>(&s.mask[a.topk[i]]), 1ull << (i / a.k));
  __syncthreads();
  if (threadIdx.x < kWave) {
    int row = 0, live = 0;
    for (int e0 = 0; e0 < a.E; e0 += kWave) {
      const int e = e0 + lane_id();
      const int n = e < a.E ? popc64(s.mask[e]) : 0;
      const int before = wave_incl_scan(n) - n;
      const uint64_t on = ballot(n > 0);
      if (e < a.E) s.first[e] = (uint16_t)(row + before);
      if (n > 0) s.live[live + popc64(on & lanemask_lt())] = (uint16_t)e;
      row += __shfl(before + n, kWave - 1, kWave);
      live += popc64(on);
    }
    if (lane_id() == 0) s.num_live = live;
  }
  __syncthreads();
}

// The r-th token of a mask.
__device__ __forceinline__ int nth_token(uint64_t mask, int r) {
  for (int i = 0; i < r; ++i) mask &= mask - 1;
  return mask ? __builtin_ctzll(mask) : 0;
}

template <typename T>
struct mma;  // eight k values of a lane: products of a 16 x 32 by a 32 x 16 tile


// 16-bit: four columns of eight rows in 16 registers; the fragment of column c
// gathers its half-words, two rows at a time.
template <typename T>
struct mma16 {
  struct Weights {
    uint32_t r[8][2];
  };
  struct Tokens {
    uint32_t v[4];
  };
  __device__ static void column(const Weights& w, int c, uint32_t (&out)[4]) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      out[p] = __builtin_amdgcn_perm(w.r[2 * p + 1][c >> 1], w.r[2 * p][c >> 1],
                                     (c & 1) ? 0x07060302u : 0x05040100u);
  }
};
template <>
struct mma<bf16> : mma16<bf16> {
  __device__ static f32x4 run(const Tokens& x, const Weights& w, int c, f32x4 acc) {
    uint32_t b[4];
    column(w, c, b);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.v),
                                                   __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  }
};
template <>
struct mma<f16> : mma16<f16> {
  __device__ static f32x4 run(const Tokens& x, const Weights& w, int c, f32x4 acc) {
    uint32_t b[4];
    column(w, c, b);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x.v),
                                                  __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  }
};
// fp32: the eight k values go one by one; which of the 32 a lane group holds
// is free as long as tokens and weights agree.
template <>
struct mma<float> {
  struct Weights {
    float r[8][4];
  };
  struct Tokens {
    float v[8];
  };
  __device__ static f32x4 run(const Tokens& x, const Weights& w, int c, f32x4 acc) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[i], w.r[i][c], acc, 0, 0, 0);
    return acc;
  }
};

// Rows k0 .. k0 + 7 (the lane's) of columns c0 .. c0 + 3 of a [K, N] matrix.
// Rows past K and columns past N are zero.
template <typename T>
__device__ __forceinline__ void load_weights(const typename elem<T>::storage* w, int64_t K,
                                             int64_t N, int64_t k0, int64_t c0, bool inside,
                                             typename mma<T>::Weights& out) {
  typedef typename elem<T>::storage S;
  if (inside) {
#pragma unroll
    for (int i = 0; i < 8; ++i) __builtin_memcpy(out.r[i], w + (k0 + i) * N + c0, 4 * sizeof(S));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      S v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool in = k0 + i < K && c0 + c < N;
        v[c] = in ? w[(k0 + i) * N + c0 + c] : S(0);
      }
      __builtin_memcpy(out.r[i], v, sizeof(v));
    }
  }
}
template <typename T>
__device__ __forceinline__ void load_tokens(const typename elem<T>::storage* row, int64_t K,
                                            int64_t k0, typename mma<T>::Tokens& out) {
  typedef typename elem<T>::storage S;
  if (k0 + 8 <= K) {
    __builtin_memcpy(out.v, row + k0, 8 * sizeof(S));
  } else {
    S v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k0 + i < K ? row[k0 + i] : S(0);
    __builtin_memcpy(out.v, v, sizeof(v));
  }
}

// acc += rows (MT x 16 of them, `row[m]` this lane's) x columns [c0, c0 + 64)
// of MATS [K, N] matrices over this wave's k-steps in [s0, s1).
template <typename T, int MATS, int MT>
__device__ __forceinline__ void wave_tile(const typename elem<T>::storage* const (&w)[MATS],
                                          const typename elem<T>::storage* const (&row)[MT],
                                          int tiles, int64_t K, int64_t N, int64_t col, int64_t s0,
                                          int64_t s1, f32x4 (&acc)[MATS][MT][4]) {
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  const int64_t c0 = col + (lane & 15) * 4;
  const bool whole = col + kCols <= N;
  for (int64_t s = s0 + wave; s < s1; s += kWaves) {
    const int64_t k0 = s * kStep + (lane >> 4) * 8;
    const bool inside = whole && s * kStep + kStep <= K;
    typename mma<T>::Weights wt[MATS];
    typename mma<T>::Tokens xt[MT];
#pragma unroll
    for (int i = 0; i < MATS; ++i) load_weights<T>(w[i], K, N, k0, c0, inside, wt[i]);
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (m < tiles) load_tokens<T>(row[m], K, k0, xt[m]);
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (m < tiles) acc[i][m][c] = mma<T>::run(xt[m], wt[i], c, acc[i][m][c]);
  }
}

// The eight waves' sums of row tile m: thread i gets columns 2 (i & 1) of
// lane (i >> 1) & 63's four, of that lane's row i >> 7, of every matrix.
template <int MATS, int MT>
__device__ __forceinline__ void fold_waves(const f32x4 (&acc)[MATS][MT][4], int m, float* s_acc,
                                           float (&v)[MATS][2]) {
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MATS; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      f32x4 t;
#pragma unroll
      for (int c = 0; c < 4; ++c) t[c] = acc[i][m][c][r];
      *reinterpret_cast<f32x4*>(s_acc + (((wave * MATS + i) * 4 + r) * kWave + lane) * 4) = t;
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MATS; ++i) {
    v[i][0] = v[i][1] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float* p = s_acc + (w * MATS + i) * 4 * kWave * 4 + threadIdx.x * 2;
      v[i][0] += p[0];
      v[i][1] += p[1];
    }
  }
}

__device__ __forceinline__ float few_gelu(float x) {
  return 0.5f * x * (1.f + erff(x * 0.70710678f));
}

// hidden = act(x W1[, x W2]), one tile of 64 hidden columns of one expert at a
// time; the waves share the reduction over d.
template <typename T, bool SWIGLU, int MT>
__global__ void __launch_bounds__(kThreads) few_up_kernel(FewArgs a) {
  typedef typename elem<T>::storage S;
  constexpr int MATS = SWIGLU ? 2 : 1;
  __shared__ Plan s_plan;
  __shared__ __attribute__((aligned(16))) float s_acc[kWaves * MATS * kRowsMma * kCols];
  make_plan(a, s_plan);
  const int lane = lane_id();
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < a.T * a.k; i += kThreads) {
      const int e = a.topk[i], t = i / a.k;
      a.inv[i] = s_plan.first[e] + popc64(s_plan.mask[e] & ((1ull << t) - 1));
    }
  }
  const int64_t per = ceil_div(a.f, (int64_t)kCols), steps = ceil_div(a.d, (int64_t)kStep);
  const int64_t items = s_plan.num_live * per;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int e = s_plan.live[item / per];
    const int64_t col = item % per * kCols;
    const uint64_t mask = s_plan.mask[e];
    const int rows = popc64(mask), tiles = (rows + kRowsMma - 1) / kRowsMma;
    const S* row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = m * kRowsMma + (lane & 15);
      row[m] = static_cast<const S*>(a.x) + (int64_t)nth_token(mask, r < rows ? r : 0) * a.d;
    }
    const S* w[MATS];
    w[0] = static_cast<const S*>(a.w1) + (int64_t)e * a.d * a.f;
    if constexpr (SWIGLU) w[1] = static_cast<const S*>(a.w2) + (int64_t)e * a.d * a.f;
    f32x4 acc[MATS][MT][4];
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][m][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    wave_tile<T, MATS, MT>(w, row, tiles, a.d, a.f, col, 0, steps, acc);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= tiles) break;
      float v[MATS][2];
      fold_waves<MATS, MT>(acc, m, s_acc, v);
      const int src = (threadIdx.x >> 1) & 63;
      const int r = m * kRowsMma + (src >> 4) * 4 + (threadIdx.x >> 7);
      const int64_t c = col + (src & 15) * 4 + (threadIdx.x & 1) * 2;
      if (r < rows) {
        S* h = static_cast<S*>(a.hidden) + (int64_t)(s_plan.first[e] + r) * a.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float z;
          if constexpr (SWIGLU) z = v[0][j] / (1.f + __expf(-v[0][j])) * v[1][j];
          else z = few_gelu(v[0][j]);
          if (c + j < a.f) h[c + j] = elem<T>::store(z);
        }
      }
    }
  }
}

// partial[s] = hidden W3 over the s-th part of f, one tile of 64 columns of
// one expert at a time.
template <typename T, int MT>
__global__ void __launch_bounds__(kThreads) few_down_kernel(FewArgs a) {
  typedef typename elem<T>::storage S;
  __shared__ Plan s_plan;
  __shared__ __attribute__((aligned(16))) float s_acc[kWaves * kRowsMma * kCols];
  make_plan(a, s_plan);
  const int lane = lane_id();
  const int64_t per = ceil_div(a.d, (int64_t)kCols), steps = ceil_div(a.f, (int64_t)kStep);
  const int64_t items = s_plan.num_live * per * a.splits;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int split = (int)(item % a.splits);
    const int64_t tile = item / a.splits;
    const int e = s_plan.live[tile / per];
    const int64_t col = tile % per * kCols;
    const int rows = popc64(s_plan.mask[e]), tiles = (rows + kRowsMma - 1) / kRowsMma;
    const int64_t first = s_plan.first[e];
    const S* row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = m * kRowsMma + (lane & 15);
      row[m] = static_cast<const S*>(a.hidden) + (first + (r < rows ? r : 0)) * a.f;
    }
    const S* w[1] = {static_cast<const S*>(a.w3) + (int64_t)e * a.f * a.d};
    f32x4 acc[1][MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[0][m][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    wave_tile<T, 1, MT>(w, row, tiles, a.f, a.d, col, steps * split / a.splits,
                        steps * (split + 1) / a.splits, acc);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= tiles) break;
      float v[1][2];
      fold_waves<1, MT>(acc, m, s_acc, v);
      const int src = (threadIdx.x >> 1) & 63;
      const int r = m * kRowsMma + (src >> 4) * 4 + (threadIdx.x >> 7);
      const int64_t c = col + (src & 15) * 4 + (threadIdx.x & 1) * 2;
      if (r < rows) {
        float* p = a.partial + ((int64_t)split * a.T * a.k + first + r) * a.d;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (c + j < a.d) p[c + j] = v[0][j];
      }
    }
  }
}

// out_t = sum_j gates_tj sum_s partial[s][inv_tj].
template <typename T>
__global__ void __launch_bounds__(256) few_combine_kernel(FewArgs a) {
  const int t = blockIdx.y;
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.d) return;
  const int64_t stride = (int64_t)a.T * a.k * a.d;
  float sum = 0.f;
  for (int j = 0; j < a.k; ++j) {
    const float* p = a.partial + (int64_t)a.inv[t * a.k + j] * a.d + c;
    float y = 0.f;
    for (int s = 0; s < a.splits; ++s) y += p[s * stride];
    sum = fmaf(a.gates[t * a.k + j], y, sum);
  }
  static_cast<typename elem<T>::storage*>(a.out)[(int64_t)t * a.d + c] = elem<T>::store(sum);
}

// Parts of the down projection's reduction: as many as give every slot a tile,
// each with a k-step for every wave.
int32_t few_splits(int64_t T, int32_t k, int32_t E, int64_t d, int64_t f) {
  const int64_t tiles = std::min<int64_t>(T * k, E) * ceil_div(d, (int64_t)kCols);
  const int64_t most = std::max<int64_t>(1, ceil_div(f, (int64_t)kStep) / kWaves);
  return (int32_t)std::max<int64_t>(1, std::min(most, kSlots / std::max<int64_t>(1, tiles)));
}

struct Layout {
  size_t inv, hidden, partial, bytes;
};
Layout few_layout(int dtype, int64_t T, int32_t k, int32_t E, int64_t d, int64_t f) {
  Layout l;
  const size_t A = (size_t)T * k;
  l.inv = 0;
  l.hidden = (size_t)round_up((int64_t)A * 4, 256);
  l.partial = l.hidden + (size_t)round_up((int64_t)(A * f) * dtype_bytes(dtype), 256);
  l.bytes = l.partial + (size_t)few_splits(T, k, E, d, f) * A * d * 4;
  return l;
}

int check_few(int dtype, int64_t T, int32_t E, int32_t k, int64_t d, int64_t f) {
  if (dtype != NT_F32 && dtype != NT_F16 && dtype != NT_BF16) return NT_ERR_DTYPE;
  if (T < 0 || E < 1 || k < 1 || k > E || k > kMaxTopK || d < 1 || f < 1) return NT_ERR_INVALID_ARG;
  if (E > NT_MAX_EXPERTS) return NT_ERR_TOO_MANY_EXPERTS;
  if (T > kMaxTokens || d > (1 << 22) || f > (1 << 22)) return NT_ERR_TOO_LARGE;
  return NT_OK;
}

template <typename T, int MT>
void launch_few(const FewArgs& a, hipStream_t stream) {
  const int64_t most = std::min<int64_t>((int64_t)a.T * a.k, a.E);
  hipLaunchKernelGGL((few_route_kernel<T>), dim3((unsigned)a.T), dim3(kRouteThreads), 0, stream, a);
  const dim3 up((unsigned)std::min<int64_t>(kSlots, most * ceil_div(a.f, (int64_t)kCols)));
  if (a.w2 != nullptr)
    hipLaunchKernelGGL((few_up_kernel<T, true, MT>), up, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((few_up_kernel<T, false, MT>), up, dim3(kThreads), 0, stream, a);
  const dim3 down(
      (unsigned)std::min<int64_t>(kSlots, most * ceil_div(a.d, (int64_t)kCols) * a.splits));
  hipLaunchKernelGGL((few_down_kernel<T, MT>), down, dim3(kThreads), 0, stream, a);
  hipLaunchKernelGGL((few_combine_kernel<T>), dim3((unsigned)ceil_div(a.d, (int64_t)256), (unsigned)a.T),
                     dim3(256), 0, stream, a);
}

template <typename T>
void launch_few(const FewArgs& a, hipStream_t stream) {
  // tokens an expert can have at most, in row tiles
  if (a.T <= kRowsMma) launch_few<T, 1>(a, stream);
  else if (a.T <= 2 * kRowsMma) launch_few<T, 2>(a, stream);
  else launch_few<T, 4>(a, stream);
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

size_t nt_moe_few_tokens_workspace_bytes(int dtype, int64_t T, int32_t E, int32_t k, int64_t d,
                                         int64_t f) {
  if (check_few(dtype, T, E, k, d, f) != NT_OK || T == 0) return 0;
  return few_layout(dtype, T, k, E, d, f).bytes;
}

int nt_moe_few_tokens(int dtype, const void* x, const float* router, const float* logits,
                      const void* w_up, const void* w_val, const void* w_down, int64_t T,
                      int32_t E, int32_t k, int64_t d, int64_t f, float* gates, int32_t* topk,
                      void* out, void* ws, size_t ws_bytes, hipStream_t stream) {
  const int st = check_few(dtype, T, E, k, d, f);
  if (st != NT_OK || T == 0) return st;
  if (x == nullptr || (router == nullptr) == (logits == nullptr) || w_up == nullptr ||
      w_down == nullptr || gates == nullptr || topk == nullptr || out == nullptr)
    return NT_ERR_INVALID_ARG;
  const Layout l = few_layout(dtype, T, k, E, d, f);
  if (ws == nullptr || ws_bytes < l.bytes || reinterpret_cast<uintptr_t>(ws) % 16 != 0)
    return NT_ERR_WORKSPACE;
  char* base = static_cast<char*>(ws);
  FewArgs a = {};
  a.x = x, a.router = router, a.logits = logits, a.w1 = w_up, a.w2 = w_val, a.w3 = w_down;
  a.T = (int32_t)T, a.E = E, a.k = k, a.d = d, a.f = f;
  a.splits = few_splits(T, k, E, d, f);
  a.gates = gates, a.topk = topk, a.out = out;
  a.inv = reinterpret_cast<int32_t*>(base + l.inv);
  a.hidden = base + l.hidden;
  a.partial = reinterpret_cast<float*>(base + l.partial);
  if (dtype == NT_F32) launch_few<float>(a, stream);
  else if (dtype == NT_F16) launch_few<f16>(a, stream);
  else launch_few<bf16>(a, stream);
  return launch_status();
}

}  // extern "C"
