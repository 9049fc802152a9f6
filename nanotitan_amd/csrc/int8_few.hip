// Products of few rows with 8-bit weights, and a whole MoE layer for the few
// tokens of a decode step on them.
//
// An expert's weights are read once for each 16, 32 or 64 of its rows (by the mean of all
// experts: stream_row_tiles), so an even batch of few rows is one read of the weights.
// They go from memory straight into the registers of the matrix instruction (their
// blocks are its operands, 1 KiB on end for a wave); the waves of a workgroup share
// a column group's reduction and add their integer sums in LDS. Sums of integers are
// exact, so neither the split nor the batch shows in a result. HBM bounds it: 128 rows of
// 8 experts, 4,096 to two times 14,336 (940 MB) 138 to 150 us, 6.3 to 6.8 TB/s where a
// read alone reaches 7.1; one row, 4,096 to 14,336, 12 us. A batch that gathers at few
// experts reads theirs again, from the caches (128 experts of 2,048 x 768, 2,048 rows:
// 51 us, half of them at one expert 56, all 28; 8 of 4,096 x 14,336, 192 rows: 98, 99, 49).
//
// A few short rows are brought to integers by every workgroup for itself, in LDS: a
// launch that did it would take longer than all of the product.
//
// The layer: routing and the tokens' integers (a workgroup a token); the up
// projections with the activation; the hidden rows' integers; the down projection;
// the gate-weighted sum. For a few tokens both roundings are the products' own, and
// who finishes the last expert's part of a column sums it.
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
// The gate-weighted sum in the down projection: what its last workgroup for a part of
// the columns needs. Of `arrived` a counter a part, zero at the start.
struct Arrive {
  const float* gates;
  const int32_t* inv;
  void* out;  // [T, N] of the hidden rows' type
  int32_t* arrived;
  int32_t T, k;
};
struct NoArrive {};

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
  __device__ __forceinline__ void load_weights(const int8_t* const (&wp)[MATS], int kb) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int t = 0; t < CT; ++t)
          w[u][i][t] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(
              wp[i] + (int64_t)(kb + u) * (kInt8Block * kInt8Block) + t * 1024));
  }
  // xp: this lane's pieces, `step` bytes a block apart; in LDS or memory.
  template <typename P>
  __device__ __forceinline__ void load_rows(const P (&xp)[MT], int step, int kb) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        x[u][m] = *reinterpret_cast<const i32x4*>(xp[m] + (int64_t)(kb + u) * step);
  }
  template <typename P>
  __device__ __forceinline__ void load(const int8_t* const (&wp)[MATS], const P (&xp)[MT],
                                       int step, int kb) {
    load_weights(wp, kb);
    load_rows(xp, step, kb);
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

constexpr int kOwnRows = 8;  // rows that a workgroup brings to integers itself, at most

// `rows` rows of f values to integers and scales in LDS, by the WAVES waves of a
// workgroup, as many a row as there are: codes[k / 64][g][held][k % 16]. row(r):
// where row r begins. Ends with a barrier.
template <typename X, int WAVES, typename F>
__device__ __forceinline__ void own_integers(F&& row, int rows, int64_t f, int held, char* codes,
                                             uint32_t* s_most, float* s_scale) {
  const int chunks = (int)(int8_pitch(f) / kVec), wave = threadIdx.x / kWave;
  const int share = rows < WAVES ? WAVES / rows : 1;  // waves of a row
  for (int r0 = 0; r0 < rows; r0 += WAVES) {
    const int r = r0 + wave / share, c0 = wave % share * kWave + lane_id();
    const bool live = r < rows;
    Some<X> v;
    uint32_t m = 0;
    if (live)
      for (int c = c0; c < chunks; c += share * kWave) {
        v.load(row(r), (int64_t)c * kVec, f);
        const uint32_t most = v.most();
        m = most > m ? most : m;
      }
#pragma unroll
    for (int o = kWave / 2; o >= 1; o >>= 1) m = max(m, (uint32_t)__shfl_xor(m, o, kWave));
    __syncthreads();  // the rows before, or the item before, are read no more
    if (lane_id() == 0) s_most[wave] = m;
    __syncthreads();
    if (!live) continue;
    for (int i = 0; i < share; ++i) m = max(m, s_most[wave / share * share + i]);
    const float s = int8_scale(m), inv = int8_inverse(s);
    if (c0 == 0) s_scale[r] = s;
    const bool once = chunks <= share * kWave;  // then v still holds it
    for (int c = c0; c < chunks; c += share * kWave) {
      if (!once) v.load(row(r), (int64_t)c * kVec, f);
      *reinterpret_cast<typename Some<X>::Codes*>(codes + (c * held + r) * 16) = v.codes(s, inv);
    }
  }
  __syncthreads();
}

// CT of the four operands of a column group, up to 16 MT rows of one expert, for
// the KW waves of a workgroup at a time. X: the rows' values, of which `held` (at
// most kOwnRows) rows an item come to integers here; or int8_t, integers.
template <typename T, typename X, int EPI, int MT, int CT, int KW, int U, bool CHOSEN,
          bool ARRIVE>
__global__ void __launch_bounds__(KW* kWave)
    int8_stream_kernel(Int8Gemm a, std::conditional_t<CHOSEN, Chosen, NoChoice> chosen,
                       std::conditional_t<ARRIVE, Arrive, NoArrive> arrive, int held) {
  typedef typename elem<T>::storage S;
  constexpr int MATS = EPI == kInt8SwiGLU ? 2 : 1, kRows = 16 * MT;
  constexpr bool kOwn = !std::is_same<X, int8_t>::value;
  static_assert(!kOwn || MT == 1, "a row tile's integers in LDS");
  extern __shared__ __attribute__((aligned(16))) char s_codes[];
  __shared__ uint32_t s_most[KW];
  __shared__ float s_scale[kOwnRows];
  __shared__ int32_t s_last;
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
    if constexpr (CHOSEN) {
      row0 = s_plan.first[e] + done;
      rows = min(popc64(s_plan.mask[e]) - done, kRows);
    } else {
      int64_t r0, r1;
      int8_expert_rows(a, e, r0, r1);
      row0 = r0 + done;
      rows = (int)(r1 - row0 < kRows ? r1 - row0 : kRows);
    }
    auto x_row = [&](int r) -> int64_t {  // of the item's row r
      if constexpr (CHOSEN) return nth_token(s_plan.mask[e], done + r);
      else return row0 + r;
    };
    const int8_t* wp[MATS];
#pragma unroll
    for (int i = 0; i < MATS; ++i)
      wp[i] = (i == 0 ? a.w : a.w2) + (e * groups + group) * kInt8Block * pitch + t0 * 1024 +
              lane * 16;
    // this wave's blocks, a stage ahead in flight; the first and the columns' scales
    // before anything is waited for
    int kb = blocks * wave / KW;
    const int kb1 = blocks * (wave + 1) / KW;
    Stage<MATS, CT, MT, U> s0, s1;
    if (kOwn && kb + U <= kb1) s0.load_weights(wp, kb);
    float sw[MATS][4];
    static_assert(CT <= KW, "a wave for each operand's columns at the end");
    const int64_t n_mine =
        group * kInt8Block + 16 * (lane >> 4) + 4 * (t0 + (wave < CT ? wave : 0));
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        sw[i][q] = n_mine + q < a.N ? (i == 0 ? a.w_scales : a.w2_scales)[e * a.N + n_mine + q] : 0.f;
    if constexpr (kOwn) {
      rows = min(rows, held);  // (what the caller promised)
      own_integers<X, KW>(
          [&](int r) {
            return static_cast<const typename elem<X>::storage*>(a.values) + x_row(r) * a.K;
          },
          rows, a.K, held, s_codes, s_most, s_scale);
    }
    std::conditional_t<kOwn, const char*, const int8_t*> xp[MT];
    const int step = kOwn ? 64 * held : 1024;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = m * 16 + (lane & 15), in = r < rows ? r : 0;
      if constexpr (kOwn) xp[m] = s_codes + ((lane >> 4) * held + in) * 16;
      else xp[m] = a.x + int8_row(x_row(in), pitch) + (lane >> 4) * 256;
    }
    i32x4 acc[MATS][CT][MT];
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][t][m] = i32x4{0, 0, 0, 0};
    if (kb + U <= kb1) {
      if (!kOwn) s0.load_weights(wp, kb);
      s0.load_rows(xp, step, kb);
      kb += U;
      for (; kb + 2 * U <= kb1; kb += 2 * U) {
        s1.load(wp, xp, step, kb);
        s0.multiply(acc);
        s0.load(wp, xp, step, kb + U);
        s1.multiply(acc);
      }
      const bool more = kb + U <= kb1;
      if (more) s1.load(wp, xp, step, kb);
      s0.multiply(acc);
      if (more) {
        s1.multiply(acc);
        kb += U;
      }
    }
    for (; kb < kb1; ++kb) {
      Stage<MATS, CT, MT, 1> s;
      s.load(wp, xp, step, kb);
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
      if (const int t = wave; t < CT) {
        const int64_t n = n_mine;
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
        const float sx = kOwn ? s_scale[r & (kOwnRows - 1)] : a.x_scales[x_row(r)];
        const int64_t at = (row0 + r) * a.N;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (n + q >= a.N) break;
          S o;
          float o2, o3;
          const float p = (float)sum[0][q] * sw[0][q] * sx;
          const float p2 = MATS == 2 ? (float)sum[MATS - 1][q] * sw[MATS - 1][q] * sx : 0.f;
          int8_epilogue<T, EPI>(p, p2, o, o2, o3);
          if constexpr (ARRIVE)  // through the L2s: the workgroups run on any XCD
            __hip_atomic_store(static_cast<float*>(a.out) + at + n + q, p, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
          else
            static_cast<S*>(a.out)[at + n + q] = o;
          if (EPI != kInt8Plain && a.out2 != nullptr) {
            a.out2[at + n + q] = o2;
            if (EPI == kInt8SwiGLU) a.out3[at + n + q] = o3;
          }
        }
      }
    }
    if constexpr (ARRIVE) {
      // The stores above went past the L2s and are complete when their wave's vmcnt is
      // zero; the counter follows that, and who counts last reads past the L2s too. A
      // fence would write back all of an L2 instead.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const int loads = s_plan.pref[a.E];
      if (threadIdx.x == 0) s_last = atomicAdd(&arrive.arrived[part], 1) == loads - 1;
      __syncthreads();
      if (s_last == 0) continue;
      const int cols = 16 * CT;
      for (int i = threadIdx.x; i < arrive.T * cols; i += blockDim.x) {
        const int t = i / cols, c = i - t * cols, j4 = c / 4 % CT;
        const int64_t n = group * kInt8Block + 16 * (c / (4 * CT)) + 4 * (t0 + j4) + c % 4;
        if (n >= a.N) continue;
        float sum = 0.f;
        for (int j = 0; j < arrive.k; ++j) {
          const float* y = static_cast<const float*>(a.out) +
                           (int64_t)arrive.inv[t * arrive.k + j] * a.N + n;
          sum = fmaf(arrive.gates[t * arrive.k + j],
                     __hip_atomic_load(y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), sum);
        }
        if constexpr (kOwn)
          static_cast<typename elem<X>::storage*>(arrive.out)[t * a.N + n] = rounded<X>(sum);
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
// What a launch's workgroups are, by the column groups that all experts have.
template <typename F>
void by_columns(int64_t groups, int row_tiles, F&& f) {
  if (groups >= (row_tiles == 4 ? 128 : 512)) f(constant<4>(), constant<4>(), constant<1>());
  else if (groups >= 128) f(constant<2>(), constant<4>(), constant<1>());
  else f(constant<1>(), constant<8>(), constant<2>());
}

template <typename T, int EPI, bool CHOSEN, typename C>
void launch_stream(const Int8Gemm& a, int64_t experts, const C& chosen, hipStream_t s) {
  const int mt = stream_row_tiles(a.A, a.E);
  const int64_t groups = int8_groups(a.N);
  // every load but an expert's last is full
  const int64_t loads = std::min<int64_t>(a.A, experts + a.A / (16 * mt));
  auto by_rows = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    by_columns(experts * groups, MT, [&](auto ct, auto kw, auto u) {
      constexpr int CT = decltype(ct)::value, KW = decltype(kw)::value;
      hipLaunchKernelGGL(
          (int8_stream_kernel<T, int8_t, EPI, MT, CT, KW, decltype(u)::value, CHOSEN, false>),
          dim3((unsigned)std::min<int64_t>(loads * groups * (4 / CT), 1 << 20)), dim3(KW * kWave),
          0, s, a, chosen, NoArrive(), 0);
    });
  };
  if (mt == 1) by_rows(constant<1>());
  else if (mt == 2) by_rows(constant<2>());
  else by_rows(constant<4>());
}

// Rows of `width` values that workgroups bring to integers themselves: up to eight, and
// 16,384 values in all, four passes of 256 lanes and 16 KiB of LDS. A launch of its own
// for them takes 4 us and the gap before the next (a layer of 512 x 2,048 for one token:
// 19.5 us for 22.5; one row, 4,096 to 14,336: 13.6 for 14.2).
bool own_rows(int64_t rows, int64_t width) {
  return rows <= kOwnRows && rows * int8_pitch(width) <= 16384;
}

// The product of at most kOwnRows rows from their values (a.values, of type X).
template <typename T, typename X, int EPI, bool CHOSEN, bool ARRIVE, typename C, typename R>
void launch_own(const Int8Gemm& a, int64_t experts, int64_t loads, int held, const C& chosen,
                const R& arrive, hipStream_t s) {
  const int64_t groups = int8_groups(a.N);
  by_columns(experts * groups, 1, [&](auto ct, auto kw, auto u) {
    constexpr int CT = decltype(ct)::value, KW = decltype(kw)::value;
    hipLaunchKernelGGL(
        (int8_stream_kernel<T, X, EPI, 1, CT, KW, decltype(u)::value, CHOSEN, ARRIVE>),
        dim3((unsigned)(loads * groups * (4 / CT))), dim3(KW * kWave), held * int8_pitch(a.K), s,
        a, chosen, arrive, held);
  });
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
  int8_t* codes;  // of the tokens; null: not written
  float* scales;
  int32_t* arrived;  // counters to clear, `parts` of them (or null)
  int32_t parts;
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
  if (a.arrived != nullptr && t == 0)
    for (int i = threadIdx.x; i < a.parts; i += kRouteThreads) a.arrived[i] = 0;
  for (int64_t c = threadIdx.x * 4; c < (a.codes == nullptr ? 0 : a.d); c += kRouteThreads * 4) {
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
  for (int64_t c = threadIdx.x * 4; c < (a.codes == nullptr ? 0 : pitch);
       c += kRouteThreads * 4) {
    const X4 v = four(c);
    int q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = int8_code(elem<T>::load(v[j]), s, inv);
    *reinterpret_cast<uint32_t*>(a.codes + int8_row(t, pitch) + c / 16 * 256 + c % 16) =
        pack_bytes(q[0], q[1], q[2], q[3]);
  }
  if (threadIdx.x == 0 && a.codes != nullptr) a.scales[t] = s;
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
  static_cast<typename elem<T>::storage*>(out)[t * d + c] = rounded<T>(sum);
}

struct Layout {
  size_t inv, offsets, arrived, x, x_scales, hidden, codes, scales, y, bytes;
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
  l.arrived = take(4 * int8_groups(d) * 4);
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

bool launch_int8_own(const Int8Gemm& a, int epi, int dtype, hipStream_t s) {
  if (!own_rows(a.A, a.K)) return false;
  const int64_t experts = std::min<int64_t>(a.E, a.A);
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    auto go = [&](auto epilogue) {
      launch_own<T, T, decltype(epilogue)::value, false, false>(a, experts, experts, (int)a.A,
                                                                NoChoice(), NoArrive(), s);
    };
    if (epi == kInt8Plain) go(constant<kInt8Plain>());
    else if (epi == kInt8SwiGLU) go(constant<kInt8SwiGLU>());
    else go(constant<kInt8Gelu>());
  });
  return true;
}

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
  Int8Gemm down = {};
  down.offsets = c.offsets, down.w = w_down, down.w_scales = down_scales;
  down.E = E, down.A = A, down.K = f, down.N = d, down.out = base + l.y;
  float* y = reinterpret_cast<float*>(base + l.y);
  if (own_rows(T, d) && own_rows(T, f)) {
    // 16 arrivals on a counter cost less than a launch, many do not
    const bool sum_here = experts <= 16;
    r.codes = nullptr;
    if (sum_here) {
      r.arrived = reinterpret_cast<int32_t*>(base + l.arrived);
      r.parts = (int32_t)(4 * int8_groups(d));
    }
    up.values = x, down.values = up.out;
    int8_by_type(dtype, [&](auto type) {
      typedef typename decltype(type)::type V;
      hipLaunchKernelGGL((int8_route_kernel<V>), dim3((unsigned)T), dim3(kRouteThreads), 0,
                         stream, r);
      if (w_val != nullptr)
        launch_own<V, V, kInt8SwiGLU, true, false>(up, experts, experts, (int)T, c, NoArrive(),
                                                   stream);
      else
        launch_own<V, V, kInt8Gelu, true, false>(up, experts, experts, (int)T, c, NoArrive(),
                                                 stream);
      if (sum_here) {
        Arrive sum = {gates, c.inv, out, r.arrived, (int32_t)T, k};
        launch_own<float, V, kInt8Plain, false, true>(down, experts, experts, (int)T, NoChoice(),
                                                      sum, stream);
      } else {
        launch_own<float, V, kInt8Plain, false, false>(down, experts, experts, (int)T,
                                                       NoChoice(), NoArrive(), stream);
        hipLaunchKernelGGL((int8_combine_kernel<V>),
                           dim3((unsigned)ceil_div(d, (int64_t)256), (unsigned)T), dim3(256), 0,
                           stream, y, c.inv, gates, k, d, out);
      }
    });
    return launch_status();
  }
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
  down.x = codes, down.x_scales = scales;
  launch_stream<float, kInt8Plain, false>(down, experts, NoChoice(), stream);
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type V;
    hipLaunchKernelGGL((int8_combine_kernel<V>),
                       dim3((unsigned)ceil_div(d, (int64_t)256), (unsigned)T), dim3(256), 0,
                       stream, y, c.inv, gates, k, d, out);
  });
  return launch_status();
}

}  // extern "C"
