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
// them at once on the matrix cores. Two launches (the up projections with the
// activation; the down projection), with one before them where the routing is
// long and one behind where many partial sums are to be added.
//
// Weights are [K, N] row-major and the matrix instruction wants each lane's
// eight k values of one column in a register quad. A lane loads eight rows of
// four neighbouring columns straight from memory and transposes them with byte
// permutes (one per two values): nothing but the tokens is read twice, nothing
// goes through LDS but the waves' partial sums at the end.
//
// Measured on MI355X (a read of 2 GiB: 7.1 TB/s): 16 tokens of 4,096, 8 experts
// of 14,336, bf16: up 285 us (6.6 TB/s), down 141 (6.7), all 433; 64 tokens: all
// 455 (6.2); 33 tokens of 2,048, 128 experts of 768, top-8, fp16:
// up 59 (6.0), down 58 (6.1), routing 7, gate sum 5, all 129; one token of 512,
// 16 experts of 2,048: 9 + 8, all 17.2 (its 12.6 MB would take 1.8: launches
// and a chain of about ten dependent memory latencies).
#include <algorithm>
#include <type_traits>

#include "bits.hpp"
#include "common.hpp"
#include "gelu.hpp"

namespace nt {
namespace {

constexpr int kMaxTokens = NT_FEW_TOKENS_MAX;
// Waves of a workgroup whose tiles take KW waves each: small workgroups fill the
// registers of a CU better (12 waves of 156 registers fit, or one workgroup of 8).
constexpr int group_waves(int tile_waves) { return tile_waves > 4 ? tile_waves : 4; }
constexpr int kMaxTileWaves = 8;
constexpr int kCols = 64;   // columns of a tile: 16 lanes x 4
constexpr int kRowsMma = 16;
constexpr int kStep = 32;   // weight rows a wave takes at a time

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Load;

// Routing in a launch of its own, or in every workgroup of the up projection.
enum { kRouteApart = 0, kRouteFused = 1, kRouteSmall = 2 };

struct FewArgs {
  const void* x;        // [T, d]
  const float* router;  // [E, d], or null
  const float* logits;  // [T, E], used without a router
  const void *w1, *w2;  // [E, d, f]; w2 null for gelu
  const void* w3;       // [E, f, d]
  int32_t T, E, k, splits;
  int32_t most_live;  // experts that can have tokens, at most
  int32_t most_loads;  // and the loads (below) that they can make
  int32_t route;      // where the routing is done
  bool arrive;        // gate sum in the down projection
  int64_t d, f;
  float* gates;       // [T, k]
  int32_t* topk;      // [T, k]
  void* out;          // [T, d]
  int32_t* arrived;   // [ceil(d / 64)]: finished parts of the columns' tiles
  int32_t* inv;       // [T, k]: row of an assignment in hidden and partial
  Load* loads;        // [1 + most_loads]
  void* hidden;       // [T k, f]
  float* partial;     // [splits][T k][d]
};

// ------------------------------------------------------------------ routing

// Choices in the order of nt_route_topk as one unsigned key, the larger first:
// the value's bits as an ordered integer (-0 as +0, every NaN below -inf), then
// the lower expert. 0: no choice.
__device__ __forceinline__ uint64_t choice_key(float z, int e) {
  uint32_t u = __float_as_uint(z);  // integers only: denormals keep their order
  if (u == 0x80000000u) u = 0u;
  const uint32_t ordered =
      (u & 0x7fffffffu) > 0x7f800000u ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
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

// This wave's part of the sums x[i] . w[i] over the columns [c0, c1), four a
// lane at a time, all N sums' loads of 512 columns in flight together. Past c1
// a lane reads the last four again and counts none twice.
template <typename T, int N>
__device__ __forceinline__ void dot_part(const typename elem<T>::storage* const (&x)[N],
                                         const float* const (&w)[N], int64_t c0, int64_t c1,
                                         float (&sum)[N]) {
  typedef typename elem<T>::storage S;
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = 0.f;
  if (c1 - c0 < 4) {
    if (c0 + lane_id() < c1)
      for (int i = 0; i < N; ++i)
        sum[i] = elem<T>::load(x[i][c0 + lane_id()]) * w[i][c0 + lane_id()];
  } else {
    typedef float W4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef S X4 __attribute__((ext_vector_type(4), aligned(sizeof(S))));
    for (int64_t b = c0; b < c1; b += 2 * kWave * 4) {
      W4 wv[2][N];
      X4 xv[2][N];
      int skip[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t c = b + (h * kWave + lane_id()) * 4, at = c + 4 <= c1 ? c : c1 - 4;
        skip[h] = c - at < 4 ? (int)(c - at) : 4;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          wv[h][i] = *reinterpret_cast<const W4*>(w[i] + at);
          xv[h][i] = *reinterpret_cast<const X4*>(x[i] + at);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sum[i] = j >= skip[h] ? fmaf(elem<T>::load(xv[h][i][j]), wv[h][i][j], sum[i]) : sum[i];
    }
  }
#pragma unroll
  for (int o = kWave / 2; o >= 1; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += __shfl_xor(sum[i], o, kWave);
}

// One token a workgroup: its logits (each wave an expert, or a part of one's
// columns where there are fewer experts than waves), then the top-k by one
// wave.
constexpr int kRouteThreads = 1024;
constexpr int kRouteWaves = kRouteThreads / kWave;
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) few_route_kernel(FewArgs a) {
  typedef typename elem<T>::storage S;
  __shared__ float s_logit[NT_MAX_EXPERTS];
  __shared__ float s_part[kRouteWaves];
  const int t = blockIdx.x, lane = lane_id(), wave = threadIdx.x / kWave;
  if (a.router != nullptr) {
    const S* x = static_cast<const S*>(a.x) + (int64_t)t * a.d;
    int parts = 1;
    while (2 * parts * a.E <= kRouteWaves) parts *= 2;
    const int64_t width = round_up(ceil_div(a.d, (int64_t)parts), 4);
    constexpr int N = 4;
    for (int i0 = wave; i0 < a.E * parts; i0 += N * kRouteWaves) {
      const int64_t c0 = i0 % parts * width, c1 = c0 + width < a.d ? c0 + width : a.d;
      const S* xs[N];
      const float* ws[N];
      float sum[N];
#pragma unroll
      for (int q = 0; q < N; ++q) {  // (with parts > 1 there is one each)
        const int i = i0 + q * kRouteWaves < a.E * parts ? i0 + q * kRouteWaves : i0;
        xs[q] = x;
        ws[q] = a.router + (int64_t)(i / parts) * a.d;
      }
      dot_part<T, N>(xs, ws, c0, c1, sum);
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const int i = i0 + q * kRouteWaves;
        if (lane == 0 && i < a.E * parts) (parts > 1 ? s_part : s_logit)[i] = sum[q];
      }
    }
    if (parts > 1) {
      __syncthreads();
      if ((int)threadIdx.x < a.E) {
        float sum = 0.f;
        for (int p = 0; p < parts; ++p) sum += s_part[threadIdx.x * parts + p];
        s_logit[threadIdx.x] = sum;
      }
    }
  } else {
    for (int e = threadIdx.x; e < a.E; e += kRouteThreads)
      s_logit[e] = a.logits[(int64_t)t * a.E + e];
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

// The same for all tokens in one workgroup of the up projection, which every
// workgroup repeats: worth it while it costs less than the launch (4.7 us and
// its gap) that it saves. A choice's place is the number of logits ahead of
// it, so that no selection waits for another: s_topk and s_value [T k].
constexpr int kFusedLogits = 512;
template <typename T, int N>
__device__ __forceinline__ void router_here(const FewArgs& a, float* s_logit) {
  typedef typename elem<T>::storage S;
  const int n = a.T * a.E, waves = blockDim.x / kWave;
  for (int i0 = threadIdx.x / kWave; i0 < n; i0 += N * waves) {
    const S* xs[N];
    const float* ws[N];
    float sum[N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int i = i0 + q * waves < n ? i0 + q * waves : i0;
      xs[q] = static_cast<const S*>(a.x) + (int64_t)(i / a.E) * a.d;
      ws[q] = a.router + (int64_t)(i % a.E) * a.d;
    }
    dot_part<T, N>(xs, ws, 0, a.d, sum);
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (lane_id() == 0 && i0 + q * waves < n) s_logit[i0 + q * waves] = sum[q];
  }
}
template <typename T>
__device__ __forceinline__ void logits_here(const FewArgs& a, float* s_logit) {
  if (a.router == nullptr) {
    for (int i = threadIdx.x; i < a.T * a.E; i += blockDim.x) s_logit[i] = a.logits[i];
  } else if (a.T * a.E * kWave <= 2 * (int)blockDim.x) {
    router_here<T, 2>(a, s_logit);
  } else {
    router_here<T, 4>(a, s_logit);
  }
  __syncthreads();
}
__device__ __forceinline__ void route_here(const FewArgs& a, const float* s_logit, int32_t* s_topk,
                                           float* s_value) {
  const int n = a.T * a.E;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int t = i / a.E, e = i - t * a.E;
    const uint64_t key = choice_key(s_logit[i], e);
    int ahead = 0;
    for (int o = 0; o < a.E; ++o) ahead += choice_key(s_logit[t * a.E + o], o) > key;
    if (ahead < a.k) {
      s_topk[t * a.k + ahead] = e;
      s_value[t * a.k + ahead] = s_logit[i];
    }
  }
  __syncthreads();
  if (blockIdx.x != 0) return;
  for (int i = threadIdx.x; i < a.T * a.k; i += blockDim.x) {
    const float* v = s_value + i / a.k * a.k;
    float den = 0.f;
    for (int j = 0; j < a.k; ++j) den += expf(v[j] - v[0]);
    a.gates[i] = expf(s_value[i] - v[0]) * (1.f / den);
    a.topk[i] = s_topk[i];
  }
}

// ------------------------------------------------------------- expert tiles

// Which tokens each expert has, the first row of each (rows by expert, then
// token) and the loads: an expert's tokens, `most_rows` at a time, so that the
// workgroups of a load hold all its sums. An expert with more tokens is read
// once for each of its loads, by different workgroups.
constexpr int kPartShift = 10;  // a load as 16 bits: expert, part
constexpr int kMaxLoads = NT_MAX_EXPERTS + kMaxTokens * kMaxTopK / kRowsMma;
static_assert(NT_MAX_EXPERTS <= 1 << kPartShift, "a load in 16 bits");
struct Plan {
  uint64_t mask[NT_MAX_EXPERTS];
  uint16_t first[NT_MAX_EXPERTS];
  uint16_t load[kMaxLoads];
  int32_t num_loads;
};

// The same for the down projection, in memory: the number of loads, then each
// one's {expert, first row, rows, 0}.
struct Load {
  int32_t expert, first, rows, pad;
};

__device__ __forceinline__ void make_plan(const FewArgs& a, const int32_t* topk, int most_rows,
                                          Plan& s) {
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) s.mask[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * a.k; i += blockDim.x)
    atomicOr(reinterpret_cast<unsigned long long*>(&s.mask[topk[i]]), 1ull << (i / a.k));
  __syncthreads();
  if (threadIdx.x < kWave) {
    int row = 0, loads = 0;
    for (int e0 = 0; e0 < a.E; e0 += kWave) {
      const int e = e0 + lane_id();
      const int n = e < a.E ? popc64(s.mask[e]) : 0, parts = (n + most_rows - 1) / most_rows;
      const int before = wave_incl_scan(n) - n, ahead = wave_incl_scan(parts) - parts;
      if (e < a.E) s.first[e] = (uint16_t)(row + before);
      for (int p = 0; p < parts; ++p)
        s.load[loads + ahead + p] = (uint16_t)(e | p << kPartShift);
      row += __shfl(before + n, kWave - 1, kWave);
      loads += __shfl(ahead + parts, kWave - 1, kWave);
    }
    if (lane_id() == 0) s.num_loads = loads;
  }
  __syncthreads();
}

// What the down projection reads of it, and its counters cleared.
__device__ __forceinline__ void write_plan(const FewArgs& a, const int32_t* topk, int most_rows,
                                           const Plan& s) {
  for (int i = threadIdx.x; i < a.T * a.k; i += blockDim.x) {
    const int e = topk[i], t = i / a.k;
    a.inv[i] = s.first[e] + popc64(s.mask[e] & ((1ull << t) - 1));
  }
  for (int i = threadIdx.x; i < s.num_loads; i += blockDim.x) {
    const int e = s.load[i] & ((1 << kPartShift) - 1);
    const int done = (s.load[i] >> kPartShift) * most_rows;
    a.loads[1 + i] = {e, s.first[e] + done, min(popc64(s.mask[e]) - done, most_rows), 0};
  }
  if (threadIdx.x == 0) a.loads[0] = {s.num_loads, 0, 0, 0};
  for (int i = threadIdx.x; i < ceil_div(a.d, (int64_t)kCols); i += blockDim.x) a.arrived[i] = 0;
}

// The same for at most eight tokens and 64 experts, by every wave on its own and
// in registers (lane e: expert e), with one barrier where the plan in LDS takes
// six: latency is all that such a call costs.
constexpr int kSmallTokens = 8;
struct SmallPlan {
  uint32_t mask, first;  // of expert lane_id()
  uint64_t live;

  __device__ __forceinline__ void make(const FewArgs& a, const float* s_logit, int32_t* s_topk,
                                       float* s_value) {
    const int e = lane_id();
    const bool writer = blockIdx.x == 0 && threadIdx.x < kWave;
    mask = 0;
    for (int t = 0; t < a.T; ++t) {
      const float z = e < a.E ? s_logit[t * a.E + e] : 0.f;
      const uint64_t key = e < a.E ? choice_key(z, e) : 0ull;
      const uint32_t lo = (uint32_t)key, hi = (uint32_t)(key >> 32);
      int ahead = 0;
      for (int o = 0; o < a.E; ++o) {
        const uint64_t other = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, o) << 32) |
                               (uint32_t)__builtin_amdgcn_readlane(lo, o);
        ahead += other > key;
      }
      if (e < a.E && ahead < a.k) {
        mask |= 1u << t;
        if (writer) {
          s_topk[t * a.k + ahead] = e;
          s_value[t * a.k + ahead] = z;
        }
      }
    }
    const int n = __popc(mask);
    first = (uint32_t)(wave_incl_scan(n) - n);
    live = ballot(n > 0);
    if (!writer) return;
    lds_wave_sync();
    for (int i = lane_id(); i < ((a.T * a.k + kWave - 1) & -kWave); i += kWave) {
      const bool in = i < a.T * a.k;
      const int t = in ? i / a.k : 0, c = in ? s_topk[i] : 0;
      const uint32_t its_first = __shfl(first, c, kWave), its_mask = __shfl(mask, c, kWave);
      if (!in) continue;
      const float* v = s_value + t * a.k;
      float den = 0.f;
      for (int j = 0; j < a.k; ++j) den += expf(v[j] - v[0]);
      a.gates[i] = expf(s_value[i] - v[0]) * (1.f / den);
      a.topk[i] = c;
      a.inv[i] = (int32_t)its_first + __popc(its_mask & ((1u << t) - 1));
    }
    if (n > 0) a.loads[1 + popc64(live & lanemask_lt())] = {e, (int32_t)first, n, 0};
    if (lane_id() == 0) a.loads[0] = {popc64(live), 0, 0, 0};
    for (int i = lane_id(); i < ceil_div(a.d, (int64_t)kCols); i += kWave) a.arrived[i] = 0;
  }
  // The i-th live expert (uniform).
  __device__ __forceinline__ int expert(int i) const {
    uint64_t m = live;
    for (; i > 0; --i) m &= m - 1;
    return __builtin_ctzll(m);
  }
};

// The r-th token of a mask.
__device__ __forceinline__ int nth_token(uint64_t mask, int r) {
  for (int i = 0; i < r; ++i) mask &= mask - 1;
  return mask ? __builtin_ctzll(mask) : 0;
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// A buffer of raw words from a uniform address.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000);
}
constexpr int kNonTemporal = 2;  // the instruction's nt bit

// Eight k values of a lane: what the matrix instructions of a step take.
// 16-bit: four columns of eight rows in 16 registers; the fragment of column c
// gathers its half-words, two rows at a time.
template <typename T>
struct mma {
  struct Weights {
    uint32_t r[8][2];
  };
  struct Tokens {
    uint32_t v[4];
  };
  __device__ static void load_row(__amdgpu_buffer_rsrc_t b, uint32_t off, uint32_t (&out)[2]) {
    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, kNonTemporal);
    out[0] = v[0], out[1] = v[1];
  }
  __device__ static void load_eight(__amdgpu_buffer_rsrc_t b, uint32_t off, uint32_t (&out)[4]) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = v[i];
  }
  __device__ static f32x4 run(const Tokens& x, const Weights& w, int c, f32x4 acc) {
    uint32_t b[4];
#pragma unroll
    for (int p = 0; p < 4; ++p)
      b[p] = __builtin_amdgcn_perm(w.r[2 * p + 1][c >> 1], w.r[2 * p][c >> 1],
                                   (c & 1) ? 0x07060302u : 0x05040100u);
    if constexpr (std::is_same<T, bf16>::value)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.v),
                                                     __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    else
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
  __device__ static void load_row(__amdgpu_buffer_rsrc_t b, uint32_t off, float (&out)[4]) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, kNonTemporal);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __uint_as_float(v[i]);
  }
  __device__ static void load_eight(__amdgpu_buffer_rsrc_t b, uint32_t off, float (&out)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(b, off, h * 16, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) out[h * 4 + i] = __uint_as_float(v[i]);
    }
  }
  __device__ static f32x4 run(const Tokens& x, const Weights& w, int c, f32x4 acc) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[i], w.r[i][c], acc, 0, 0, 0);
    return acc;
  }
};

// A tile of 64 columns of [K, N] matrices: its first column, and the lane's
// first. The last tile of a width reaches back to be whole (its first columns
// are then another tile's too and not stored); in matrices of fewer than 64
// columns, lanes past the end repeat the last four.
struct TileColumns {
  int64_t start;
  uint32_t lane;
  TileColumns() = default;
  __device__ __forceinline__ TileColumns(int64_t col, int64_t N) {
    start = col + kCols <= N ? col : N > kCols ? N - kCols : 0;
    const int64_t c = (lane_id() & 15) * 4, most = N - start - 4;
    lane = (uint32_t)(c <= most || most < 0 ? c : most);
  }
};

// Four columns of eight weight rows for each of MATS matrices, and eight
// values of each of TL tokens, as a lane holds them for one step.
template <typename T, int MATS, int TL>
struct Step {
  typedef typename elem<T>::storage S;
  typename mma<T>::Weights w[MATS];
  typename mma<T>::Tokens x[TL];

  // Buffer loads: the step's first row goes into the scalar base and the lane's
  // eight offsets (bytes, the same for every step and matrix) stay 32-bit: as
  // 64-bit addresses they took 32 registers more. `left` rows remain from the
  // step's first; those past them are out of the buffer's range and read as
  // zero. The weights are read once (non-temporal).
  __device__ __forceinline__ void load_weights(const S* const (&base)[MATS], int64_t N,
                                               const TileColumns (&tc)[MATS], int64_t step,
                                               int64_t left, const uint32_t (&off)[8]) {
#pragma unroll
    for (int i = 0; i < MATS; ++i) {
      const int64_t size = (left * N - tc[i].start) * (int64_t)sizeof(S);
      const auto buf = buffer_of(base[i] + step * kStep * N + tc[i].start,
                                 size < 0xffffffffll ? (uint32_t)size : 0xffffffffu);
#pragma unroll
      for (int r = 0; r < 8; ++r) mma<T>::load_row(buf, off[r], w[i].r[r]);
    }
  }
  template <int MT>
  __device__ __forceinline__ void load_tokens(const S* x0, const uint32_t (&row)[MT],
                                              int64_t step) {
    const auto buf = buffer_of(x0 + step * kStep, 0xffffffffu);
#pragma unroll
    for (int m = 0; m < TL; ++m) mma<T>::load_eight(buf, row[m], x[m].v);
  }
  // Past the last whole step: `left` values of each token.
  template <int MT>
  __device__ __forceinline__ void load_last_tokens(const S* x0, const uint32_t (&row)[MT],
                                                   int64_t step, int64_t left) {
    const int k0 = (lane_id() >> 4) * 8;
#pragma unroll
    for (int m = 0; m < TL; ++m) {
      S v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        v[r] = k0 + r < left ? x0[row[m] / sizeof(S) + step * kStep + r] : S(0);
      __builtin_memcpy(x[m].v, v, sizeof(v));
    }
  }
  // Layers with a width of less than four: element by element, in both of their
  // projections.
  __device__ __forceinline__ void load_narrow_weights(const S* const (&base)[MATS], int64_t N,
                                                      const TileColumns (&tc)[MATS],
                                                      int64_t step, int64_t left) {
    const int k0 = (lane_id() >> 4) * 8;
#pragma unroll
    for (int i = 0; i < MATS; ++i) {
      const int64_t c0 = tc[i].start + (lane_id() & 15) * 4;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        S v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          v[c] = k0 + r < left && c0 + c < N ? base[i][(step * kStep + k0 + r) * N + c0 + c] : S(0);
        __builtin_memcpy(w[i].r[r], v, sizeof(v));
      }
    }
  }
  template <int MT>
  __device__ __forceinline__ void multiply(f32x4 (&acc)[MATS][MT][4]) const {
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int m = 0; m < TL; ++m) acc[i][m][c] = mma<T>::run(x[m], w[i], c, acc[i][m][c]);
  }
};

// acc += TL x 16 token rows (byte row[m] of x0, this lane's) times the tile,
// over the k-steps [s0, s1): the tile's KW waves take them in turn, each with
// the next step's loads in flight while it multiplies.
template <int TL, int KW, bool NARROW, typename T, int MATS, int MT>
__device__ __forceinline__ void wave_tile(const typename elem<T>::storage* const (&base)[MATS],
                                          const typename elem<T>::storage* x0,
                                          const uint32_t (&row)[MT],
                                          const TileColumns (&tc)[MATS], int64_t K, int64_t N,
                                          int64_t s0, int64_t s1,
                                          f32x4 (&acc)[MATS][MT][4]) {
  typedef Step<T, MATS, TL> Held;
  int64_t s = s0 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave % KW);
  if constexpr (NARROW) {
    for (; s < s1; s += KW) {
      Held t;
      t.load_narrow_weights(base, N, tc, s, K - s * kStep);
      t.load_last_tokens(x0, row, s, K - s * kStep);
      t.multiply(acc);
    }
    return;
  }
  uint32_t off[8];
#pragma unroll
  for (int r = 0; r < 8; ++r)
    off[r] = (((uint32_t)(lane_id() >> 4) * 8 + r) * (uint32_t)N + tc[0].lane) *
             (uint32_t)sizeof(typename elem<T>::storage);
  const int64_t whole = s1 < K / kStep ? s1 : K / kStep;
  const int n = s < whole ? (int)((whole - s + KW - 1) / KW) : 0;
  auto load = [&](Held& t, int i) {
    const int64_t at = s + (int64_t)i * KW;
    t.load_weights(base, N, tc, at, K - at * kStep, off);
    t.load_tokens(x0, row, at);
  };
  // The loads of the loop are unconditional: behind a branch, the wait for an
  // older step's registers would be for the newer ones too. (Two steps in
  // flight beside the one multiplied: 143 -> 179 us for 33 tokens, 128 experts
  // of 2,048 x 768.)
  Held t0, t1;
  if constexpr (sizeof(typename elem<T>::storage) == 4 && TL * MATS >= 4) {
    // float32 weights and these many sums fill the registers: one step at a time
    for (int i = 0; i < n; ++i) {
      load(t0, i);
      t0.multiply(acc);
    }
  } else if (n > 0) {
    load(t0, 0);
    int i = 1;
    for (; i + 1 < n; i += 2) {
      load(t1, i);
      t0.multiply(acc);
      load(t0, i + 1);
      t1.multiply(acc);
    }
    if (i < n) load(t1, i);
    t0.multiply(acc);
    if (i < n) t1.multiply(acc);
  }
  s += (int64_t)n * KW;
  if (s < s1) {
    Held t;
    t.load_weights(base, N, tc, s, K - s * kStep, off);
    t.load_last_tokens(x0, row, s, K - s * kStep);
    t.multiply(acc);
  }
}

// The same for any number of row tiles up to MT (none: zeros).
template <int KW, bool NARROW, typename T, int MATS, int MT>
__device__ __forceinline__ void wave_tiles(int tiles,
                                           const typename elem<T>::storage* const (&base)[MATS],
                                           const typename elem<T>::storage* x0,
                                           const uint32_t (&row)[MT],
                                           const TileColumns (&tc)[MATS], int64_t K, int64_t N,
                                           int64_t s0, int64_t s1,
                                           f32x4 (&acc)[MATS][MT][4]) {
#pragma unroll
  for (int i = 0; i < MATS; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][m][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (tiles == 1) wave_tile<1, KW, NARROW, T>(base, x0, row, tc, K, N, s0, s1, acc);
  if constexpr (MT >= 2)
    if (tiles == 2) wave_tile<2, KW, NARROW, T>(base, x0, row, tc, K, N, s0, s1, acc);
  if constexpr (MT == 4)
    if (tiles > 2) wave_tile<4, KW, NARROW, T>(base, x0, row, tc, K, N, s0, s1, acc);
}

// The sums of a tile's KW waves for row tile m. A thread gets 16 / KW columns
// of one row (fold_row, fold_col) for every matrix; a wave alone with its tile
// keeps its own, four columns of four rows.
template <int KW, int MATS, int MT>
__device__ __forceinline__ void fold_waves(const f32x4 (&acc)[MATS][MT][4], int m, float* s_acc,
                                           float (&v)[MATS][16 / KW]) {
  constexpr int N = 16 / KW;
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  if constexpr (KW == 1) {
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) v[i][r * 4 + c] = acc[i][m][c][r];
  } else {
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
    const float* s = s_acc + wave / KW * KW * MATS * 1024 + threadIdx.x % (KW * kWave) * N;
#pragma unroll
    for (int i = 0; i < MATS; ++i) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[i][j] = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int j = 0; j < N; ++j) v[i][j] += s[(w * MATS + i) * 1024 + j];
    }
  }
}
// Where value j of a thread lies: the row of row tile m and the column of the
// matrix. The tile's sums are [4][64 lanes][4 columns], lane l's rows 4 (l / 16).
template <int KW>
__device__ __forceinline__ int fold_row(int m, int j) {
  const int at = KW == 1 ? j / 4 * 256 + lane_id() * 4 : threadIdx.x % (KW * kWave) * (16 / KW);
  return m * kRowsMma + (at >> 2 & 63) / 16 * 4 + at / 256;
}
template <int KW, bool NARROW>
__device__ __forceinline__ int64_t fold_col(const TileColumns& tc, int64_t N, int j) {
  const int at = KW == 1 ? j / 4 * 256 + lane_id() * 4 + j % 4
                         : threadIdx.x % (KW * kWave) * (16 / KW) + j;
  const int64_t c = (at >> 2 & 15) * 4, most = N - tc.start - 4;
  return tc.start + (NARROW || c <= most ? c : most) + (at & 3);
}

// hidden = act(x W1[, x W2]), one tile of 64 hidden columns of one expert (or
// HALVES = 2 neighbouring ones of a single matrix: as much in flight a wave as
// with two matrices) for KW waves at a time.
template <typename T, bool SWIGLU, int HALVES, int MT, int KW, bool NARROW>
__global__ void __launch_bounds__(group_waves(KW) * kWave) few_up_kernel(FewArgs a) {
  typedef typename elem<T>::storage S;
  constexpr int MATS = SWIGLU ? 2 : HALVES, N = 16 / KW;
  constexpr int kWaves = group_waves(KW), kTiles = kWaves / KW;
  __shared__ Plan s_plan;
  __shared__ __attribute__((aligned(16))) float
      s_acc[KW == 1 ? 3 * kFusedLogits : kWaves * MATS * kRowsMma * kCols];
  const int lane = lane_id();
  const bool small = KW == kMaxTileWaves && a.route == kRouteSmall;
  constexpr int kRows = MT * kRowsMma;
  static_assert(kSmallTokens <= kRows, "a small plan's experts are one load each");
  SmallPlan here = {};
  int num_loads;
  if (small) {
    logits_here<T>(a, s_acc);
    here.make(a, s_acc, reinterpret_cast<int32_t*>(s_acc + kFusedLogits), s_acc + 2 * kFusedLogits);
    num_loads = popc64(here.live);
  } else {
    const int32_t* topk = a.topk;
    if (a.route == kRouteFused) {
      int32_t* s_topk = reinterpret_cast<int32_t*>(s_acc + kFusedLogits);
      logits_here<T>(a, s_acc);
      route_here(a, s_acc, s_topk, s_acc + 2 * kFusedLogits);
      topk = s_topk;
    }
    make_plan(a, topk, kRows, s_plan);
    if (blockIdx.x == 0) write_plan(a, topk, kRows, s_plan);
    num_loads = s_plan.num_loads;
  }
  const int64_t per = ceil_div(a.f, (int64_t)kCols * HALVES), steps = ceil_div(a.d, (int64_t)kStep);
  const int64_t items = num_loads * per;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave / KW);
  for (int64_t first = (int64_t)blockIdx.x * kTiles; first < items;
       first += (int64_t)gridDim.x * kTiles) {
    // past the last tile, a group repeats it and stores nothing
    const int64_t item = first + group < items ? first + group : items - 1;
    const int load = __builtin_amdgcn_readfirstlane(small ? here.expert((int)(item / per))
                                                         : s_plan.load[item / per]);
    const int e = load & ((1 << kPartShift) - 1), done = (load >> kPartShift) * kRows;
    const int64_t col = item % per * HALVES * kCols;
    TileColumns tc[MATS];
#pragma unroll
    for (int i = 0; i < MATS; ++i) tc[i] = TileColumns(col + i * (HALVES - 1) * kCols, a.f);
    uint64_t mask = small ? (uint32_t)__builtin_amdgcn_readlane(here.mask, e) : s_plan.mask[e];
    const int first_row =
        done + (small ? __builtin_amdgcn_readlane(here.first, e) : (int)s_plan.first[e]);
    for (int i = 0; i < done; ++i) mask &= mask - 1;  // the tokens of its earlier loads
    const int rows = __builtin_amdgcn_readfirstlane(min(popc64(mask), kRows));
    const S* w[MATS];
    w[0] = static_cast<const S*>(a.w1) + (int64_t)e * a.d * a.f;
    if constexpr (MATS == 2)
      w[1] = static_cast<const S*>(SWIGLU ? a.w2 : a.w1) + (int64_t)e * a.d * a.f;
    S* hidden = static_cast<S*>(a.hidden) + (int64_t)first_row * a.f;
    const int tiles = (rows + kRowsMma - 1) / kRowsMma;
    uint32_t row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = m * kRowsMma + (lane & 15);
      row[m] = ((uint32_t)nth_token(mask, r < rows ? r : 0) * (uint32_t)a.d + (lane >> 4) * 8) *
               (uint32_t)sizeof(S);
    }
    f32x4 acc[MATS][MT][4];
    wave_tiles<KW, NARROW, T>(tiles, w, static_cast<const S*>(a.x), row, tc, a.d, a.f, 0, steps,
                              acc);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if ((kTiles == 1 || KW == 1) && m >= tiles) break;
      float v[MATS][N];
      fold_waves<KW, MATS, MT>(acc, m, s_acc, v);
      if (item != first + group) continue;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int r = fold_row<KW>(m, j);
          const int64_t c = fold_col<KW, NARROW>(tc[h], a.f, j);
          float z;
          if constexpr (SWIGLU) z = v[0][j] / (1.f + __expf(-v[0][j])) * v[1][j];
          else {
            float bell;
            z = v[h][j] * gelu_cdf<T>(v[h][j], bell);
          }
          if (r < rows && c >= col + h * kCols && c < a.f)
            hidden[(int64_t)r * a.f + c] = to_bits<T>(z);
        }
    }
  }
}

// out_t = sum_j gates_tj sum_s partial[s][inv_tj], column c of token t. SHARED:
// written by workgroups of this launch.
template <typename T, bool SHARED>
__device__ __forceinline__ void combine_at(const FewArgs& a, int t, int64_t c) {
  const int64_t stride = (int64_t)a.T * a.k * a.d;
  float sum = 0.f;
#pragma unroll 4
  for (int j = 0; j < a.k; ++j) {
    const float* p = a.partial + (int64_t)a.inv[t * a.k + j] * a.d + c;
    float y = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s)
      y += SHARED ? __hip_atomic_load(p + s * stride, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                  : p[s * stride];
    sum = fmaf(a.gates[t * a.k + j], y, sum);
  }
  static_cast<typename elem<T>::storage*>(a.out)[(int64_t)t * a.d + c] = to_bits<T>(sum);
}

template <typename T>
__global__ void __launch_bounds__(256) few_combine_kernel(FewArgs a) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c < a.d) combine_at<T, false>(a, blockIdx.y, c);
}

// partial[s] = hidden W3 over the s-th part of f, one tile of 64 columns of
// one expert for KW waves at a time. Where a workgroup has a tile alone (KW =
// 8) and at most one, whoever finishes the last part of a tile's columns also
// sums them over the experts: partials are written and read through the L2s
// (agent scope: the workgroups run on any XCD); a wave's are complete when its
// vmcnt is zero, and the counter is touched behind the barrier after that.
// Elsewhere a launch of its own sums them: with eight tiles a workgroup the
// waits cost 30 us of 90 (33 tokens, 128 experts of 768 x 2,048).
template <typename T, int HALVES, int MT, int KW, bool NARROW>
__global__ void __launch_bounds__(group_waves(KW) * kWave) few_down_kernel(FewArgs a) {
  typedef typename elem<T>::storage S;
  constexpr int kWaves = group_waves(KW), kTiles = kWaves / KW, N = 16 / KW;
  __shared__ __attribute__((aligned(16))) float
      s_acc[KW == 1 ? 4 : kWaves * HALVES * kRowsMma * kCols];
  __shared__ int32_t s_last;
  const int lane = lane_id();
  const int64_t per = ceil_div(a.d, (int64_t)kCols * HALVES), steps = ceil_div(a.f, (int64_t)kStep);
  const int64_t most = (int64_t)a.most_loads * per * a.splits;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave / KW);
  for (int64_t start = (int64_t)blockIdx.x * kTiles; start < most;
       start += (int64_t)gridDim.x * kTiles) {
    // the entry and the number of entries in one wait: past the number it is
    // arbitrary, but there
    const int64_t at = start + group < most ? start + group : most - 1;
    const int num_loads = __builtin_amdgcn_readfirstlane(a.loads[0].expert);
    Load ld = a.loads[1 + at / a.splits / per];
    const int64_t items = num_loads * per * a.splits;
    if (start >= items) return;
    const bool mine = start + group < items;
    const int64_t item = mine ? start + group : items - 1;
    if (!mine) ld = a.loads[num_loads];
    ld.expert = __builtin_amdgcn_readfirstlane(ld.expert);
    ld.first = __builtin_amdgcn_readfirstlane(ld.first);
    const int rows = __builtin_amdgcn_readfirstlane(ld.rows);
    const int split = (int)(item % a.splits);
    const int64_t tile = item / a.splits % per, col = tile * HALVES * kCols;
    TileColumns tc[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) tc[h] = TileColumns(col + h * kCols, a.d);
    const S* hidden = static_cast<const S*>(a.hidden) + (int64_t)ld.first * a.f;
    const S* w[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
      w[h] = static_cast<const S*>(a.w3) + (int64_t)ld.expert * a.f * a.d;
    float* out = a.partial + ((int64_t)split * a.T * a.k + ld.first) * a.d;
    const int tiles = (rows + kRowsMma - 1) / kRowsMma;
    uint32_t row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = m * kRowsMma + (lane & 15);
      row[m] = ((uint32_t)(r < rows ? r : 0) * (uint32_t)a.f + (lane >> 4) * 8) *
               (uint32_t)sizeof(S);
    }
    f32x4 acc[HALVES][MT][4];
    wave_tiles<KW, NARROW, T>(tiles, w, hidden, row, tc, a.f, a.d, steps * split / a.splits,
                              steps * (split + 1) / a.splits, acc);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if ((kTiles == 1 || KW == 1) && m >= tiles) break;
      float v[HALVES][N];
      fold_waves<KW, HALVES, MT>(acc, m, s_acc, v);
      if (!mine) continue;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int r = fold_row<KW>(m, j);
          const int64_t c = fold_col<KW, NARROW>(tc[h], a.d, j);
          if (r >= rows || c < col + h * kCols || c >= a.d) continue;
          float* p = out + (int64_t)r * a.d + c;
          if (KW == 8 && HALVES == 1 && a.arrive)
            __hip_atomic_store(p, v[h][j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          else
            *p = v[h][j];
        }
    }
    if (KW == 8 && HALVES == 1 && a.arrive) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (threadIdx.x == 0) s_last = atomicAdd(&a.arrived[tile], 1) == num_loads * a.splits - 1;
      __syncthreads();
      if (s_last && col + lane < a.d)
        for (int t = threadIdx.x / kWave; t < a.T; t += kWaves)
          combine_at<T, true>(a, t, col + lane);
    }
  }
}

// Waves that fit the chip (256 CUs) by the kernels' registers: with one row tile
// sixteen a CU, twelve for two matrices, else twelve and eight.
int64_t few_waves(int row_tiles, int mats) {
  return 256 * (16 - 4 * (mats - 1) - (row_tiles == 1 ? 0 : 4));
}

// Row tiles of a load: by the tokens that an expert has on average, since more
// take the registers that hold twice the waves. One up to four tokens (33 tokens,
// top-8 of 128: 143 -> 131 us), two up to 20 (64 tokens of top-2 of 8, 4,096 x
// 14,336: SwiGLU 473 -> 447 us, GELU 391 -> 324; with one expert in every
// token's choice, so twice loaded, 502 -> 520 and 427 -> 397).
int few_row_tiles(int64_t T, int32_t k, int32_t E) {
  if (T <= kRowsMma || T * k <= 4 * E) return 1;
  return T <= 2 * kRowsMma || T * k <= 20 * E ? 2 : 4;
}

// Loads that T k assignments make at most: none is empty, and besides each
// expert's first all follow a full one.
int32_t few_loads(int64_t T, int32_t k, int32_t E) {
  const int64_t A = T * k, rows = few_row_tiles(T, k, E) * kRowsMma;
  return (int32_t)std::min<int64_t>(A, std::min<int64_t>(A, E) + (T > rows ? A / rows : 0));
}

// Parts of the down projection's reduction: as many as give every CU the
// workgroups that it holds (two with one row tile), each with two k-steps for
// every wave (one token of 512: 17.3 us, with one k-step 17.9).
int32_t few_splits(int64_t T, int32_t k, int32_t E, int64_t d, int64_t f) {
  const int64_t tiles = std::min<int64_t>(T * k, E) * ceil_div(d, (int64_t)kCols);
  const int64_t most = std::max<int64_t>(1, ceil_div(f, (int64_t)kStep) / (2 * kMaxTileWaves));
  const int64_t slots = few_row_tiles(T, k, E) == 1 ? 512 : 256;
  return (int32_t)std::max<int64_t>(1, std::min(most, slots / std::max<int64_t>(1, tiles)));
}

// How an expert kernel's tiles lie: as many waves each as leave every tile its
// place at once. Fewer waves a tile means fewer of the folds and barriers that
// end one; with more tiles than waves a wave takes several in turn. Eight waves
// are for tiles that have a CU each: with more, some CUs have two and the others
// one, and four waves a tile share them better (4 tokens, top-8 of 64, 2,048 x
// 768: 80 -> 64 us; 6 tokens, top-2 of 16, 512 x 2,048: 35 -> 25). One matrix
// over a long reduction is taken 128 columns at a time by eight waves where
// those tiles fill whole rounds of the CUs: twice as much in flight a wave (16
// tokens, 14,336 x 4,096: 157 -> 138 us; with three steps a wave instead, 33
// tokens, 768 x 2,048, 58 -> 62).
struct FewTiles {
  int halves, waves;
  int64_t count;
};
FewTiles few_tiles(int row_tiles, int64_t experts, int64_t K, int64_t N, int64_t parts, int mats,
                   bool pairs) {
  FewTiles t = {1, kMaxTileWaves, experts * ceil_div(N, (int64_t)kCols) * parts};
  const int64_t paired = experts * ceil_div(N, (int64_t)2 * kCols) * parts;
  if (pairs && mats == 1 && K / parts >= 16 * kMaxTileWaves * kStep &&
      paired * 20 >= ceil_div(paired, 256) * 256 * 17) {
    t.halves = 2;
    t.count = paired;
  } else {
    if (t.count > 256) t.waves = kMaxTileWaves / 2;
    while (t.waves > 1 && t.count * t.waves > few_waves(row_tiles, mats)) t.waves /= 2;
  }
  return t;
}

struct Layout {
  size_t arrived, inv, loads, hidden, partial, bytes;
};
Layout few_layout(int dtype, int64_t T, int32_t k, int32_t E, int64_t d, int64_t f) {
  Layout l;
  const int64_t A = T * k;
  auto after = [](size_t at, int64_t bytes) { return at + (size_t)round_up(bytes, 256); };
  l.arrived = 0;
  l.inv = after(l.arrived, ceil_div(d, (int64_t)kCols) * 4);
  l.loads = after(l.inv, A * 4);
  l.hidden = after(l.loads, (1 + few_loads(T, k, E)) * (int64_t)sizeof(Load));
  l.partial = after(l.hidden, A * f * dtype_bytes(dtype));
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

// f(halves, waves of a tile) as constants. Two 64-column tiles side by side are
// for the 16-bit types (float32's would not fit the registers).
template <typename T, bool NARROW, typename F>
void by_tiles(const FewTiles& t, F&& f) {
  const auto one = std::integral_constant<int, 1>();
  const auto eight = std::integral_constant<int, 8>();
  if constexpr (NARROW) {
    f(one, eight);
  } else {
    if (t.halves == 2) {
      if constexpr (sizeof(typename elem<T>::storage) == 2)
        f(std::integral_constant<int, 2>(), eight);
    } else if (t.waves == 8) f(one, eight);
    else if (t.waves == 4) f(one, std::integral_constant<int, 4>());
    else if (t.waves == 2) f(one, std::integral_constant<int, 2>());
    else f(one, one);
  }
}
// A workgroup for every group_waves / KW tiles of all loads that there can be (a
// tile in a second round would cost as much as the first; those without one
// leave), up to eight on each CU: past that they take several in turn.
dim3 few_grid(const FewArgs& a, const FewTiles& t, int tile_waves) {
  const int64_t waves = group_waves(tile_waves), tiles = t.count / a.most_live * a.most_loads;
  return dim3((unsigned)std::min<int64_t>(8192 / waves, ceil_div(tiles * tile_waves, waves)));
}

template <typename T, int MT, bool NARROW>
void launch_few(FewArgs a, hipStream_t stream) {
  constexpr bool kPairs = sizeof(typename elem<T>::storage) == 2;
  // Routing inside the up projection while it is short (see route_here): at
  // most 128 comparisons a thread, and eight of the router's sums a wave
  // (with 32, in workgroups of four waves, 8 tokens took 40 us for 28).
  const int64_t n = (int64_t)a.T * a.E;
  const bool swiglu = a.w2 != nullptr;
  const FewTiles up = few_tiles(MT, a.most_live, a.d, a.f, 1, swiglu ? 2 : 1, kPairs);
  a.route = kRouteApart;
  if (n <= kFusedLogits && a.T * a.k <= kFusedLogits && n * a.E <= 1 << 16 &&
      (a.router == nullptr || (n <= 8 * up.waves && n * a.d <= 1 << 15)))
    a.route = a.T <= kSmallTokens && a.E <= kWave && up.waves == kMaxTileWaves ? kRouteSmall
                                                                               : kRouteFused;
  if (a.route == kRouteApart)
    hipLaunchKernelGGL((few_route_kernel<T>), dim3((unsigned)a.T), dim3(kRouteThreads), 0, stream,
                       a);
  by_tiles<T, NARROW>(up, [&](auto halves, auto waves) {
    constexpr int H = decltype(halves)::value, KW = decltype(waves)::value;
    const dim3 grid = few_grid(a, up, KW), block(group_waves(KW) * kWave);
    if (swiglu && H == 1)
      hipLaunchKernelGGL((few_up_kernel<T, true, 1, MT, KW, NARROW>), grid, block, 0, stream, a);
    if (!swiglu)
      hipLaunchKernelGGL((few_up_kernel<T, false, H, MT, KW, NARROW>), grid, block, 0, stream, a);
  });
  const FewTiles down = few_tiles(MT, a.most_live, a.f, a.d, a.splits, 1, kPairs);
  // 16 arrivals on a counter and the sum of a few tokens by one workgroup cost
  // less than a launch (one token of 512: 17 against 19 us); 40 arrivals, or 32
  // tokens, do not (25 against 22)
  a.arrive = down.halves == 1 && down.waves == kMaxTileWaves && a.most_live * a.splits <= 16 &&
             a.T <= kSmallTokens;
  by_tiles<T, NARROW>(down, [&](auto halves, auto waves) {
    constexpr int H = decltype(halves)::value, KW = decltype(waves)::value;
    hipLaunchKernelGGL((few_down_kernel<T, H, MT, KW, NARROW>), few_grid(a, down, KW),
                       dim3(group_waves(KW) * kWave), 0, stream, a);
  });
  if (!a.arrive)
    hipLaunchKernelGGL((few_combine_kernel<T>),
                       dim3((unsigned)ceil_div(a.d, (int64_t)256), (unsigned)a.T), dim3(256), 0,
                       stream, a);
}

template <typename T>
void launch_few(const FewArgs& a, hipStream_t stream) {
  // a lane's four columns have to exist (the loads' width)
  if (a.d < 4 || a.f < 4) launch_few<T, 4, true>(a, stream);
  else if (const int tiles = few_row_tiles(a.T, a.k, a.E); tiles == 1)
    launch_few<T, 1, false>(a, stream);
  else if (tiles == 2) launch_few<T, 2, false>(a, stream);
  else launch_few<T, 4, false>(a, stream);
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
  a.most_live = (int32_t)std::min<int64_t>(T * k, E);
  a.most_loads = few_loads(T, k, E);
  a.gates = gates, a.topk = topk, a.out = out;
  a.arrived = reinterpret_cast<int32_t*>(base + l.arrived);
  a.inv = reinterpret_cast<int32_t*>(base + l.inv);
  a.loads = reinterpret_cast<Load*>(base + l.loads);
  a.hidden = base + l.hidden;
  a.partial = reinterpret_cast<float*>(base + l.partial);
  if (dtype == NT_F32) launch_few<float>(a, stream);
  else if (dtype == NT_F16) launch_few<f16>(a, stream);
  else launch_few<bf16>(a, stream);
  return launch_status();
}

}  // extern "C"
