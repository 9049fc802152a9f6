// Products of few rows with 8-bit weights, and a whole MoE layer for the few
// tokens of a decode step on them.
//
// With at most 64 rows an expert the product is one read of the weights, so they
// go from memory straight into the registers of the matrix instruction (their
// blocks are its operands, 1 KiB on end for a wave); the waves of a workgroup share
// a column group's reduction and add their integer sums in LDS. Sums of integers are
// exact, so neither the split nor the batch shows in a result.
//
// The layer: routing and the tokens' integers (a workgroup a token); the up
// projections with the activation; the hidden rows' integers; the down projection;
// the gate-weighted sum.
#include <algorithm>
#include <type_traits>

#include "choice.hpp"
#include "int8_gemm.hpp"

namespace nt {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Rows by expert for a decode step: token t chose expert e where bit t of mask[e]
// is set; an expert's rows are its tokens in order.
struct Chosen {
  const int32_t* topk;  // [T, k]
  int32_t T, k;
  int32_t* offsets;  // [E + 1], written for the down projection
  int32_t* inv;      // [T, k]: row of an assignment
};
struct NoChoice {};

struct StreamPlan {
  int32_t pref[NT_MAX_EXPERTS + 1];  // loads of the experts before e
};
struct ChosenPlan : StreamPlan {
  uint64_t mask[NT_MAX_EXPERTS];
  int32_t first[NT_MAX_EXPERTS + 1];
};

__device__ __forceinline__ void make_chosen(const Chosen& c, int E, int rows, ChosenPlan& s) {
  for (int e = threadIdx.x; e < E; e += blockDim.x) s.mask[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < c.T * c.k; i += blockDim.x)
    atomicOr(reinterpret_cast<unsigned long long*>(&s.mask[c.topk[i]]), 1ull << (i / c.k));
  __syncthreads();
  if (threadIdx.x < kWave) {
    int row = 0, loads = 0;
    for (int e0 = 0; e0 < E; e0 += kWave) {
      const int e = e0 + lane_id();
      const int n = e < E ? popc64(s.mask[e]) : 0, l = (n + rows - 1) / rows;
      const int rn = wave_incl_scan(n), ln = wave_incl_scan(l);
      if (e < E) {
        s.first[e + 1] = row + rn;
        s.pref[e + 1] = loads + ln;
      }
      row += __shfl(rn, kWave - 1, kWave);
      loads += __shfl(ln, kWave - 1, kWave);
    }
    if (lane_id() == 0) s.first[0] = s.pref[0] = 0;
  }
  __syncthreads();
  if (blockIdx.x != 0) return;
  for (int e = threadIdx.x; e <= E; e += blockDim.x) c.offsets[e] = s.first[e];
  for (int i = threadIdx.x; i < c.T * c.k; i += blockDim.x) {
    const int e = c.topk[i];
    c.inv[i] = s.first[e] + popc64(s.mask[e] & ((1ull << (i / c.k)) - 1));
  }
}
__device__ __forceinline__ int nth_token(uint64_t mask, int r) {
  for (int i = 0; i < r; ++i) mask &= mask - 1;
  return mask ? __builtin_ctzll(mask) : 0;
}

// A stage of a wave's reduction: U blocks of MATS matrices' CT operands and of MT
// row tiles.
template <int MATS, int CT, int MT, int U>
struct Stage {
  i32x4 w[U][MATS][CT], x[U][MT];
  __device__ __forceinline__ void load(const int8_t* const (&wp)[MATS],
                                       const int8_t* const (&xp)[MT], int kb) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int t = 0; t < CT; ++t)
          w[u][i][t] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(
              wp[i] + (int64_t)(kb + u) * (kInt8Block * kInt8Block) + t * 1024));
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        x[u][m] = *reinterpret_cast<const i32x4*>(xp[m] + (int64_t)(kb + u) * 1024);
  }
  __device__ __forceinline__ void multiply(i32x4 (&acc)[MATS][CT][MT]) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int m = 0; m < MT; ++m)
            acc[i][t][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][i][t], x[u][m],
                                                                 acc[i][t][m], 0, 0, 0);
  }
};

// CT of the four operands of a column group, up to 16 MT rows of one expert, for
// the KW waves of a workgroup at a time.
template <typename T, int EPI, int MT, int CT, int KW, int U, bool CHOSEN>
__global__ void __launch_bounds__(KW* kWave)
    int8_stream_kernel(Int8Gemm a, std::conditional_t<CHOSEN, Chosen, NoChoice> chosen) {
  typedef typename elem<T>::storage S;
  constexpr int MATS = EPI == kInt8SwiGLU ? 2 : 1, kRows = 16 * MT;
  __shared__ std::conditional_t<CHOSEN, ChosenPlan, StreamPlan> s_plan;
  __shared__ __attribute__((aligned(16))) int32_t s_acc[KW * MATS * CT * kWave * 4];
  if constexpr (CHOSEN) make_chosen(chosen, a.E, kRows, s_plan);
  else int8_row_tiles(a, kRows, s_plan.pref);
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t pitch = int8_pitch(a.K), groups = int8_groups(a.N);
  const int blocks = (int)(pitch / kInt8Block);
  const int64_t parts = groups * (4 / CT), items = s_plan.pref[a.E] * parts;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int load = (int)(item / parts);
    const int64_t part = item - load * parts, group = part / (4 / CT);
    const int t0 = (int)(part % (4 / CT)) * CT;
    int lo = 0, hi = a.E - 1;  // the largest e with pref[e] <= load
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_plan.pref[mid] <= load) lo = mid;
      else hi = mid - 1;
    }
    const int e = __builtin_amdgcn_readfirstlane(lo);
    const int done = (load - s_plan.pref[e]) * kRows;
    int64_t row0;
    int rows;
    const int8_t* xp[MT];
    if constexpr (CHOSEN) {
      uint64_t mask = s_plan.mask[e];
      row0 = s_plan.first[e] + done;
      rows = min(popc64(mask) - done, kRows);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = m * 16 + (lane & 15);
        xp[m] = a.x + int8_row(nth_token(mask, done + (r < rows ? r : 0)), pitch) +
                (lane >> 4) * 256;
      }
    } else {
      int64_t r0, r1;
      int8_expert_rows(a, e, r0, r1);
      row0 = r0 + done;
      rows = (int)(r1 - row0 < kRows ? r1 - row0 : kRows);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = m * 16 + (lane & 15);
        xp[m] = a.x + int8_row(row0 + (r < rows ? r : 0), pitch) + (lane >> 4) * 256;
      }
    }
    const int8_t* wp[MATS];
#pragma unroll
    for (int i = 0; i < MATS; ++i)
      wp[i] = (i == 0 ? a.w : a.w2) + (e * groups + group) * kInt8Block * pitch + t0 * 1024 +
              lane * 16;
    i32x4 acc[MATS][CT][MT];
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][t][m] = i32x4{0, 0, 0, 0};
    // this wave's blocks, a stage ahead in flight
    int kb = blocks * wave / KW;
    const int kb1 = blocks * (wave + 1) / KW;
    if (kb + U <= kb1) {
      Stage<MATS, CT, MT, U> s0, s1;
      s0.load(wp, xp, kb);
      kb += U;
      for (; kb + 2 * U <= kb1; kb += 2 * U) {
        s1.load(wp, xp, kb);
        s0.multiply(acc);
        s0.load(wp, xp, kb + U);
        s1.multiply(acc);
      }
      const bool more = kb + U <= kb1;
      if (more) s1.load(wp, xp, kb);
      s0.multiply(acc);
      if (more) {
        s1.multiply(acc);
        kb += U;
      }
    }
    for (; kb < kb1; ++kb) {
      Stage<MATS, CT, MT, 1> s;
      s.load(wp, xp, kb);
      s.multiply(acc);
    }
    // the waves' sums, a row tile at a time; then a wave an operand's columns
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m * 16 >= rows) break;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int t = 0; t < CT; ++t)
          *reinterpret_cast<i32x4*>(s_acc + (((wave * MATS + i) * CT + t) * kWave + lane) * 4) =
              acc[i][t][m];
      __syncthreads();
      const int r = m * 16 + (lane & 15);
      for (int t = wave; t < CT; t += KW) {
        const int64_t n = group * kInt8Block + 16 * (lane >> 4) + 4 * (t0 + t);
        i32x4 sum[MATS];
#pragma unroll
        for (int i = 0; i < MATS; ++i) {
          sum[i] = i32x4{0, 0, 0, 0};
#pragma unroll
          for (int w = 0; w < KW; ++w)
            sum[i] += *reinterpret_cast<const i32x4*>(
                s_acc + (((w * MATS + i) * CT + t) * kWave + lane) * 4);
        }
        if (r >= rows) continue;
        float sx;
        if constexpr (CHOSEN) sx = a.x_scales[nth_token(s_plan.mask[e], done + r)];
        else sx = a.x_scales[row0 + r];
        const int64_t at = (row0 + r) * a.N;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (n + q >= a.N) break;
          S o[3];
          const float p = (float)sum[0][q] * a.w_scales[e * a.N + n + q] * sx;
          const float p2 =
              MATS == 2 ? (float)sum[MATS - 1][q] * a.w2_scales[e * a.N + n + q] * sx : 0.f;
          int8_epilogue<T, EPI>(p, p2, o[0], o[1], o[2]);
          static_cast<S*>(a.out)[at + n + q] = o[0];
          if (EPI != kInt8Plain && a.out2 != nullptr) {
            static_cast<S*>(a.out2)[at + n + q] = o[1];
            if (EPI == kInt8SwiGLU) static_cast<S*>(a.out3)[at + n + q] = o[2];
          }
        }
      }
    }
  }
}

template <int V>
using constant = std::integral_constant<int, V>;

// Row tiles of a load of the weights, by the rows an expert has on average: more
// take registers and the activations' loads; fewer read the weights of an expert
// with more rows again (128 rows of 8 experts, 14,336 x 4,096: 77 us with two, 105
// with one).
int stream_row_tiles(int64_t rows, int64_t experts) {
  const int64_t mean = ceil_div(rows, experts);
  return mean <= 6 ? 1 : mean <= 20 ? 2 : 4;
}

// A workgroup takes a whole column group (four operands) for four waves where these
// fill the chip twice; half of one (a row of 4,096 to 14,336: 12.2 us, with a
// quarter 12.5) or, where there are few, a quarter for eight waves with two blocks
// each in flight (14,336 to 4,096: 11.9 us; half of one for four waves 13.8). Eight
// waves or more blocks in flight hold no more bytes in flight than the memory needs
// and leave fewer workgroups to overlap (940 MB of 8 experts' two matrices: 138 us,
// 6.8 TB/s; eight waves 153, two blocks 150, four quarters 153).
template <typename T, int EPI, bool CHOSEN, typename C>
void launch_stream(const Int8Gemm& a, int64_t experts, const C& chosen, hipStream_t s) {
  const int mt = stream_row_tiles(a.A, a.E);
  const int64_t groups = int8_groups(a.N);
  // every load but an expert's last is full
  const int64_t loads = std::min<int64_t>(a.A, experts + a.A / (16 * mt));
  auto go = [&](auto mt, auto ct, auto kw, auto u) {
    constexpr int MT = decltype(mt)::value, CT = decltype(ct)::value, KW = decltype(kw)::value;
    hipLaunchKernelGGL((int8_stream_kernel<T, EPI, MT, CT, KW, decltype(u)::value, CHOSEN>),
                       dim3((unsigned)std::min<int64_t>(loads * groups * (4 / CT), 1 << 20)),
                       dim3(KW * kWave), 0, s, a, chosen);
  };
  auto by_columns = [&](auto mt) {
    if (experts * groups >= (decltype(mt)::value == 4 ? 128 : 512))
      go(mt, constant<4>(), constant<4>(), constant<1>());
    else if (experts * groups >= 128)
      go(mt, constant<2>(), constant<4>(), constant<1>());
    else
      go(mt, constant<1>(), constant<8>(), constant<2>());
  };
  if (mt == 1) by_columns(constant<1>());
  else if (mt == 2) by_columns(constant<2>());
  else by_columns(constant<4>());
}

// ------------------------------------------------------------------ routing

struct FewRoute {
  const void* x;        // [T, d]
  const float* router;  // [E, d], or null
  const float* logits;  // [T, E], used without a router
  int32_t E, k;
  int64_t d;
  float* gates;
  int32_t* topk;
  int8_t* codes;  // [T, pitch]
  float* scales;
};

constexpr int kRouteThreads = 1024;
constexpr int kRouteWaves = kRouteThreads / kWave;

// A workgroup a token: its integers, its logits (a wave an expert), the order of
// its choices (a thread an expert: its place is the number ahead of it).
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) int8_route_kernel(FewRoute a) {
  typedef typename elem<T>::storage S;
  typedef float W4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef S X4 __attribute__((ext_vector_type(4), aligned(sizeof(S))));
  __shared__ float s_logit[NT_MAX_EXPERTS];
  __shared__ uint64_t s_key[NT_MAX_EXPERTS];
  __shared__ int32_t s_expert[kMaxTopK];
  __shared__ uint32_t s_most[kRouteWaves];
  const int64_t t = blockIdx.x;
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  const S* x = static_cast<const S*>(a.x) + t * a.d;
  auto four = [&](int64_t c) {  // columns c .. c + 3, zeros past the row's end
    X4 v;
    if (c + 4 <= a.d) {
      v = *reinterpret_cast<const X4*>(x + c);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = c + j < a.d ? x[c + j] : S(0);
    }
    return v;
  };
  uint32_t m = 0;
  for (int64_t c = threadIdx.x * 4; c < a.d; c += kRouteThreads * 4) {
    const X4 v = four(c);
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, abs_bits(elem<T>::load(v[j])));
  }
#pragma unroll
  for (int o = kWave / 2; o >= 1; o >>= 1) m = max(m, (uint32_t)__shfl_xor(m, o, kWave));
  if (lane == 0) s_most[wave] = m;
  if (a.router != nullptr) {
    for (int e = wave; e < a.E; e += kRouteWaves) {
      const float* w = a.router + (int64_t)e * a.d;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      int64_t c = lane * 4;
#pragma unroll 4
      for (; c + 4 <= a.d; c += kWave * 4) {
        const W4 u = *reinterpret_cast<const W4*>(w + c);
        const X4 v = *reinterpret_cast<const X4*>(x + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = fmaf(elem<T>::load(v[j]), u[j], sum[j]);
      }
      for (; c < a.d; ++c) sum[0] = fmaf(elem<T>::load(x[c]), w[c], sum[0]);
      const float total = wave_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
      if (lane == 0) s_logit[e] = total;
    }
  } else {
    for (int e = threadIdx.x; e < a.E; e += kRouteThreads) s_logit[e] = a.logits[t * a.E + e];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRouteWaves; ++i) m = max(m, s_most[i]);
  const float s = int8_scale(m), inv = int8_inverse(s);
  const int64_t pitch = int8_pitch(a.d);
  for (int64_t c = threadIdx.x * 4; c < pitch; c += kRouteThreads * 4) {
    const X4 v = four(c);
    int q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = int8_code(elem<T>::load(v[j]), s, inv);
    *reinterpret_cast<uint32_t*>(a.codes + int8_row(t, pitch) + c / 16 * 256 + c % 16) =
        pack_bytes(q[0], q[1], q[2], q[3]);
  }
  if (threadIdx.x == 0) a.scales[t] = s;
  const int e = threadIdx.x;
  const uint64_t key = e < a.E ? choice_key(s_logit[e], e) : 0;
  if (e < a.E) s_key[e] = key;
  __syncthreads();
  if (e < a.E) {
    int ahead = 0;
    for (int o = 0; o < a.E; ++o) ahead += s_key[o] > key;
    if (ahead < a.k) s_expert[ahead] = e;
  }
  __syncthreads();
  if (wave != 0) return;
  const int mine = lane < a.k ? s_expert[lane] : s_expert[0];
  const float z = choice_value(s_key[mine]), top = choice_value(s_key[s_expert[0]]);
  const float p = lane < a.k ? expf(z - top) : 0.f;
  const float den = wave_sum(p);
  if (lane < a.k) {
    a.gates[t * a.k + lane] = p * (1.f / den);
    a.topk[t * a.k + lane] = mine;
  }
}

// out_t = sum_j gates_tj y[inv_tj].
template <typename T>
__global__ void __launch_bounds__(256) int8_combine_kernel(const float* y, const int32_t* inv,
                                                           const float* gates, int32_t k,
                                                           int64_t d, void* out) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (c >= d) return;
  float sum = 0.f;
#pragma unroll 4
  for (int j = 0; j < k; ++j)
    sum = fmaf(gates[t * k + j], y[(int64_t)inv[t * k + j] * d + c], sum);
  static_cast<typename elem<T>::storage*>(out)[t * d + c] = to_bits<T>(sum);
}

struct Layout {
  size_t inv, offsets, x, x_scales, hidden, codes, scales, y, bytes;
};
Layout layout(int dtype, int64_t T, int32_t k, int32_t E, int64_t d, int64_t f) {
  Layout l;
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (size_t)round_up(bytes, 256);
    return here;
  };
  const int64_t A = T * k;
  l.inv = take(A * 4);
  l.offsets = take((E + 1) * 4);
  l.x = take(int8_rows_bytes(T, int8_pitch(d)));
  l.x_scales = take(T * 4);
  l.hidden = take(A * f * dtype_bytes(dtype));
  l.codes = take(int8_rows_bytes(A, int8_pitch(f)));
  l.scales = take(A * 4);
  l.y = take(A * d * 4);
  l.bytes = at;
  return l;
}

int check_few(int dtype, int64_t T, int32_t E, int32_t k, int64_t d, int64_t f) {
  if (!int8_float(dtype)) return NT_ERR_DTYPE;
  if (T < 0 || E < 1 || k < 1 || k > E || k > kMaxTopK || d < 1 || f < 1) return NT_ERR_INVALID_ARG;
  if (E > NT_MAX_EXPERTS) return NT_ERR_TOO_MANY_EXPERTS;
  if (T > NT_FEW_TOKENS_MAX || d > kInt8MaxK || f > kInt8MaxK) return NT_ERR_TOO_LARGE;
  return NT_OK;
}

}  // namespace

void launch_int8_stream(const Int8Gemm& a, int epi, int dtype, hipStream_t s) {
  const int64_t experts = std::min<int64_t>(a.E, a.A);
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    if (epi == kInt8Plain) launch_stream<T, kInt8Plain, false>(a, experts, NoChoice(), s);
    else if (epi == kInt8SwiGLU) launch_stream<T, kInt8SwiGLU, false>(a, experts, NoChoice(), s);
    else launch_stream<T, kInt8Gelu, false>(a, experts, NoChoice(), s);
  });
}

}  // namespace nt

using namespace nt;

extern "C" {

size_t nt_int8_moe_few_tokens_workspace_bytes(int dtype, int64_t T, int32_t E, int32_t k,
                                              int64_t d, int64_t f) {
  if (check_few(dtype, T, E, k, d, f) != NT_OK || T == 0) return 0;
  return layout(dtype, T, k, E, d, f).bytes;
}

int nt_int8_moe_few_tokens(int dtype, const void* x, const float* router, const float* logits,
                           const int8_t* w_up, const float* up_scales, const int8_t* w_val,
                           const float* val_scales, const int8_t* w_down,
                           const float* down_scales, int64_t T, int32_t E, int32_t k, int64_t d,
                           int64_t f, float* gates, int32_t* topk, void* out, void* ws,
                           size_t ws_bytes, hipStream_t stream) {
  int st = check_few(dtype, T, E, k, d, f);
  if (st != NT_OK || T == 0) return st;
  auto bad = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  if (x == nullptr || (router == nullptr) == (logits == nullptr) || w_up == nullptr ||
      up_scales == nullptr || (w_val == nullptr) != (val_scales == nullptr) || w_down == nullptr ||
      down_scales == nullptr || gates == nullptr || topk == nullptr || out == nullptr ||
      bad(w_up) || bad(w_val) || bad(w_down))
    return NT_ERR_INVALID_ARG;
  const Layout l = layout(dtype, T, k, E, d, f);
  if (ws == nullptr || ws_bytes < l.bytes || bad(ws)) return NT_ERR_WORKSPACE;
  char* base = static_cast<char*>(ws);
  FewRoute r = {};
  r.x = x, r.router = router, r.logits = logits, r.E = E, r.k = k, r.d = d;
  r.gates = gates, r.topk = topk;
  r.codes = reinterpret_cast<int8_t*>(base + l.x);
  r.scales = reinterpret_cast<float*>(base + l.x_scales);
  Chosen c = {};
  c.topk = topk, c.T = (int32_t)T, c.k = k;
  c.offsets = reinterpret_cast<int32_t*>(base + l.offsets);
  c.inv = reinterpret_cast<int32_t*>(base + l.inv);
  const int64_t A = T * k, experts = std::min<int64_t>(A, E);
  Int8Gemm up = {};
  up.x = r.codes, up.x_scales = r.scales, up.w = w_up, up.w_scales = up_scales;
  up.w2 = w_val, up.w2_scales = val_scales;
  up.E = E, up.A = A, up.K = d, up.N = f, up.out = base + l.hidden;
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type V;
    hipLaunchKernelGGL((int8_route_kernel<V>), dim3((unsigned)T), dim3(kRouteThreads), 0, stream,
                       r);
    if (w_val != nullptr) launch_stream<V, kInt8SwiGLU, true>(up, experts, c, stream);
    else launch_stream<V, kInt8Gelu, true>(up, experts, c, stream);
  });
  int8_t* codes = reinterpret_cast<int8_t*>(base + l.codes);
  float* scales = reinterpret_cast<float*>(base + l.scales);
  st = nt_int8_rows(dtype, up.out, A, f, codes, scales, stream);
  if (st != NT_OK) return st;
  Int8Gemm down = {};
  down.x = codes, down.x_scales = scales, down.offsets = c.offsets, down.w = w_down;
  down.w_scales = down_scales;
  down.E = E, down.A = A, down.K = f, down.N = d, down.out = base + l.y;
  launch_stream<float, kInt8Plain, false>(down, experts, NoChoice(), stream);
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type V;
    hipLaunchKernelGGL((int8_combine_kernel<V>),
                       dim3((unsigned)ceil_div(d, (int64_t)256), (unsigned)T), dim3(256), 0,
                       stream, reinterpret_cast<const float*>(base + l.y), c.inv, gates, k, d, out);
  });
  return launch_status();
}

}  // extern "C"
