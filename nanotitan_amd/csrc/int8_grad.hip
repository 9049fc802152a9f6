// Gradients through frozen 8-bit weights:
//
//   dX[a, k] = sum_n dOut[a, n] w[e, n, k],   w = q s[e, n]
//
// on the 16-bit matrix cores. The weights are read as integers, a quarter of what
// bringing them to 16 bits first would read and write, and turned on the way to LDS:
// a thread's 64 bytes are 16 values of k for four neighbouring n, and it writes for
// each k its four n. (q + 128) s - 128 s as one fused multiply-add rounds q s once.
//
// Rounding weights to 16 bits is an error as large as the output's own: a product's
// gradient is off by 2.9e-4 of its norm in float16 and 2.3e-3 in bfloat16, where the
// output's rounding is 2.1e-4 and 1.7e-3, and float16 holds no weight past 65,504. So
// dOut times the scales goes in as two bfloat16 terms (2^-17) and the weights are their
// integers, exact in bfloat16: what is left is the output's rounding. Both terms meet the
// same operands in LDS, a step each, so the second costs matrix instructions but no
// weights (14,312 rows of 2,048 by 128 experts' 768: 93 us with rounded weights, 158 by
// terms with the launch that makes them; 8,192 rows of 14,336 by 8 of 4,096: 1,056 and
// 1,778). Rounded weights are the caller's choice.
//
// Through a feed-forward block there would be five such roundings: what the forward keeps
// and the epilogue are float32, and the gradient of the hidden values goes on as terms for
// the next weights.
//
// Gradients in float32 are three such terms everywhere: 24 bits. That is three 16-bit
// products where one in float32 has a 16th of their rate (8 experts of 4,096 x 14,336,
// 8,192 rows: 2.7 ms, with float32 weights 5.4).
#include <algorithm>
#include <type_traits>

#include "gemm_common.hpp"
#include "int8_gemm.hpp"

namespace nt {
namespace {

// Terms, TermsDual: from terms and the weights' integers, out for one or two matrices;
// Gelu, SwiGLU: to such terms.
enum Int8GradEpilogue { kGradPlain, kGradGelu, kGradSwiGLU, kGradTerms, kGradTermsDual };

struct Int8Grad {
  Int8Gemm rows;             // offsets, E, A; K: output columns, N: the reduction
  const void *dout, *dout2;  // [A, N] or terms; of the second matrix
  int64_t pitch;             // of dout's rows
  const float *aux, *aux2;   // gelu' or gate, value [A, K]
  const float *next, *next2;  // scales of the weights that the terms meet [E, K]
  void* terms2;
};

constexpr int64_t kGradMaxN = 1 << 22;
constexpr int kGradBM = 128, kGradWaves = 4;
constexpr int kGradThreads = kGradWaves * kWave;

// A row (a value of k) of the turned weights is 64 n, 8 chunks of 16 bytes; chunk c
// is stored at c ^ turned_swizzle(k). An operand takes rows 16 j + 4 t + m (j, m
// < 4), whose swizzles are all eight values twice: its reads touch every bank once.
__device__ __forceinline__ int turned_swizzle(int k) { return (k >> 1 & 1) | (k >> 4 & 3) << 1; }

template <typename T>
constexpr int terms_of = std::is_same<T, float>::value ? 3 : 2;

// Eight values of row `row` from column n on as TERMS planes of terms, each what those
// before leave: a value of 2^-100 or more to 2^-17 by two, 2^-25 by three. An infinity or
// a NaN is its first term and leaves nothing; a finite value's first term is finite.
template <int TERMS>
__device__ __forceinline__ void put_terms(void* terms, int64_t row, int64_t rows, int64_t pitch,
                                          int64_t n, const float* values) {
  constexpr float kInfinity = __builtin_inff(), kMost = int8_most<bf16>::value;
  float z[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = values[j];
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    uint32_t w[4];
    auto first = [&](int j) {  // (past the first term nothing is that large)
      return i == 0 && fabsf(z[j]) < kInfinity ? fminf(fmaxf(z[j], -kMost), kMost) : z[j];
    };
    auto rest = [&](int j, uint32_t term) {
      z[j] = fabsf(z[j]) < kInfinity ? z[j] - __uint_as_float(term) : 0.f;
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = pack2<bf16>(first(2 * j), first(2 * j + 1));
      rest(2 * j, w[j] << 16);
      rest(2 * j + 1, w[j] & 0xffff0000u);
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(terms) + (i * rows + row) * pitch + n) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Terms of a gradient times its experts' scales, a wave a row.
constexpr int kTermRows = 4;
template <typename T>
__global__ void __launch_bounds__(kTermRows* kWave)
    int8_terms_kernel(const void* dout, const int32_t* offsets, const float* w_scales, int32_t E,
                      int64_t A, int64_t N, void* terms) {
  const int64_t row = (int64_t)blockIdx.x * kTermRows +
                      __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (row >= A) return;
  int lo = 0, hi = E - 1;  // the last expert that begins at or before the row
  while (offsets != nullptr && lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (offsets[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  const auto* in = static_cast<const typename elem<T>::storage*>(dout) + row * N;
  const float* sc = w_scales + lo * N;
  const int64_t pitch = int8_pitch(N), end = round_up(N, (int64_t)16);
  for (int64_t n = lane_id() * 8; n < end; n += kWave * 8) {
    Some<T, 8> v;
    Some<float, 8> s;
    v.load(in, n, N);
    s.load(sc, n, N);
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = elem<T>::load(v.v[j]) * s.v[j];
    put_terms<terms_of<T>>(terms, row, A, pitch, n, z);
  }
}

// IN: dout and dout2 are terms.
template <typename T, int EPI, int BN, bool IN>
__global__ void __launch_bounds__(kGradThreads, BN == 256 ? 2 : 3) int8_grad_kernel(Int8Grad g) {
  typedef typename elem<T>::storage S;
  // terms of a value of dOut; none: rounded weights
  constexpr int TERMS = IN ? terms_of<T> : 0;
  constexpr int TURNS = TERMS > 0 ? TERMS : 1;  // steps of the same weights
  typedef std::conditional_t<(TERMS > 0), bf16, T> M;
  typedef typename mfma_op<M>::vec vec;
  const Int8Gemm& a = g.rows;
  // of a wave: 64 rows by half of the columns
  constexpr int BM = kGradBM, WGN = 2, AB = BM / 2 / 16, CG = BN / 2 / 64;
  typedef OperandTile<BM, true, 64, kGradWaves> TA;
  constexpr int kA = TA::kBytes, kB = BN * 128;
  __shared__ __attribute__((aligned(1024))) char smem[2 * kA + kB];
  __shared__ int32_t s_pref[NT_MAX_EXPERTS + 1];
  char* turned = smem + 2 * kA;
  int8_row_tiles(a, BM, s_pref);
  const int64_t all = (int64_t)__builtin_amdgcn_readfirstlane(s_pref[a.E]) * a.ntn;
  const int64_t total = all < INT32_MAX ? all : INT32_MAX;  // (more: malformed offsets)
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
  const int nk1 = (int)ceil_div(a.N, (int64_t)64), nw = EPI == kGradTermsDual ? 2 * nk1 : nk1;
  const int nk = nw * TURNS;
  TA ta;
  ta.init(g.pitch, wave, lane);
  FragReader<BM, true, AB, 64> fa;
  fa.init(wm * 64, lane);
  // of a block of 64 columns a wave turns all, or one of two waves half of each 16;
  // thread: KT values of k, four n from n0 on
  constexpr int kShare = kGradWaves * 64 / BN, KT = 16 / kShare;
  typedef uint32_t Words __attribute__((ext_vector_type(KT / 4)));
  const int block = wave / kShare, k_half = wave % kShare * KT;
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
    const int64_t kb = col0 / kInt8Block + block;  // (none past the last)
    const bool has = kb < kblocks;

    Words w[4];
    float4 s;
    auto fetch_weights = [&](int step) {
      const bool second = EPI == kGradTermsDual && step >= nk1;
      const int64_t nb = second ? step - nk1 : step;
      const int8_t* at = (second ? a.w2 : a.w) +
                         ((e * groups + nb) * kblocks + (has ? kb : kblocks - 1)) * 4096 +
                         lane * 64 + k_half;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const Words*>(at + i * 16);
      if constexpr (TERMS == 0) {
        const int64_t n = nb * 64 + n0;
        const float* sc = a.w_scales + e * a.N + n;
        if (n + 4 <= a.N) {
          typedef float V4 __attribute__((ext_vector_type(4), aligned(4)));
          const V4 v = *reinterpret_cast<const V4*>(sc);
          s = make_float4(v[0], v[1], v[2], v[3]);
        } else {
          s = make_float4(n < a.N ? sc[0] : 0.f, n + 1 < a.N ? sc[1] : 0.f,
                          n + 2 < a.N ? sc[2] : 0.f, 0.f);
        }
      }
    };
    auto fetch_rows = [&](int kt, char* lds) {
      const int step = kt / TURNS;
      const bool second = EPI == kGradTermsDual && step >= nk1;
      const int64_t nb = second ? step - nk1 : step;
      const int64_t left = round_up(a.N, (int64_t)(TERMS > 0 ? 16 : 8)) - nb * 64;
      const int64_t kv = left < 64 ? left : 64;
      const uint16_t* d = static_cast<const uint16_t*>(second ? g.dout2 : g.dout) +
                          (kt % TURNS * a.A + row0) * g.pitch + nb * 64;
      ta.issue(d, ((rows - 1) * g.pitch + kv) * 2, lds, kv, wave);
    };
    auto turn_by = [&](auto&& value) {  // value(i, q + 128): of the integer q of column i
      uint32_t u[4][KT / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < KT / 4; ++d) u[i][d] = w[i][d] ^ 0x80808080u;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = value(i, (float)(u[i][j / 4] >> (8 * (j % 4)) & 255u));
        const int k = block * 64 + 16 * g4 + k_half + j;
        *reinterpret_cast<uint2*>(turned + k * 128 +
                                  ((2 * i4 + (t4 >> 1)) ^ turned_swizzle(k)) * 16 +
                                  (t4 & 1) * 8) =
            make_uint2(pack2<M>(v[0], v[1]), pack2<M>(v[2], v[3]));
      }
    };
    auto turn = [&]() {
      if constexpr (TERMS > 0) {
        turn_by([](int, float u) { return u - 128.f; });
      } else {
        // what int8_value gives: scales whose values pass the type's largest are rare
        constexpr float kMost = int8_most<T>::value;
        const float sc[4] = {s.x, s.y, s.z, s.w};
        const bool large = sc[0] > kMost / 128 || sc[1] > kMost / 128 || sc[2] > kMost / 128 ||
                           sc[3] > kMost / 128;
        if (__any(large)) {
          turn_by([&](int i, float u) {
            const float v = (u - 128.f) * sc[i];
            return v > kMost ? kMost : v < -kMost ? -kMost : v;  // (a NaN stays one)
          });
        } else {
          turn_by([&](int i, float u) {
            return in_float32<T>(fmaf(u, sc[i], -128.f * sc[i]));
          });
        }
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
    fetch_weights(0);
    fetch_rows(0, smem);
    for (int kt = 0; kt < nk; ++kt) {
      wait_vmcnt<0>();  // this step's rows are in LDS, its weights in registers
      if (kt % TURNS == 0) turn();
      __syncthreads();
      if (kt + 1 < nk) {
        if ((kt + 1) % TURNS == 0) fetch_weights((kt + 1) / TURNS);
        fetch_rows(kt + 1, smem + (kt + 1 & 1) * kA);
      }
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
            for (int b = 0; b < AB; ++b) acc[b][c][t] = mfma_op<M>::run(y, x[b], acc[b][c][t]);
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
        if constexpr (EPI == kGradGelu || EPI == kGradSwiGLU) {
          float x1[16], x2[16], s1[16], s2[16], z1[16], z2[16];
          int8_get(g.aux + at, width, x1);
          int8_get(g.next + e * a.K + n, width, s1);
          if constexpr (EPI == kGradSwiGLU) {
            int8_get(g.aux2 + at, width, x2);
            int8_get(g.next2 + e * a.K + n, width, s2);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float d = acc[b][c][j / 4][j % 4];
            if constexpr (EPI == kGradGelu) {
              z1[j] = j < width ? d * x1[j] * s1[j] : 0.f;
            } else {
              const float z = x1[j], sg = sigmoid_of<T>(z);
              z1[j] = j < width ? d * x2[j] * sg * (1.f + z * (1.f - sg)) * s1[j] : 0.f;
              z2[j] = j < width ? d * z * sg * s2[j] : 0.f;
            }
          }
#pragma unroll
          for (int h = 0; h < 16; h += 8) {
            put_terms<terms_of<T>>(a.out, row0 + m, a.A, kpitch, n + h, z1 + h);
            if constexpr (EPI == kGradSwiGLU)
              put_terms<terms_of<T>>(g.terms2, row0 + m, a.A, kpitch, n + h, z2 + h);
          }
        } else {
          S o[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = to_bits<T>(acc[b][c][j / 4][j % 4]);
          int8_put(static_cast<S*>(a.out) + at, width, o);
        }
      }
    }
  }
}

int run_grad(int dtype, int epi, Int8Grad g, hipStream_t s) {
  Int8Gemm& a = g.rows;
  const bool terms = epi >= kGradTerms, to_terms = epi == kGradGelu || epi == kGradSwiGLU;
  if (!int8_float(dtype)) return NT_ERR_DTYPE;
  if (a.E < 1 || a.A < 0 || a.K < 1 || a.N < 1) return NT_ERR_INVALID_ARG;
  if (a.E > NT_MAX_EXPERTS) return NT_ERR_TOO_MANY_EXPERTS;
  if (a.K > kInt8MaxK || a.N > kGradMaxN || a.A > kInt8MaxRows) return NT_ERR_TOO_LARGE;
  const bool in = terms || dtype == NT_F32 || g.pitch == 0;
  if (in) g.pitch = int8_pitch(a.N);
  if (g.pitch > kGradMaxN) return NT_ERR_TOO_LARGE;  // a tile's rows within 31 bits
  if (a.A == 0) return NT_OK;
  auto bad = [](const void* p) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  const bool two = epi == kGradTermsDual;
  if (g.pitch < a.N || g.pitch % 8 != 0 || bad(g.dout) || bad(a.w) || a.out == nullptr ||
      (a.offsets == nullptr && a.E != 1) || (!in && a.w_scales == nullptr) ||
      (two && (bad(g.dout2) || bad(a.w2))) ||
      (to_terms && (g.aux == nullptr || g.next == nullptr || bad(a.out))) ||
      (epi == kGradSwiGLU && (g.aux2 == nullptr || g.next2 == nullptr || bad(g.terms2))))
    return NT_ERR_INVALID_ARG;
  const int64_t cus = device_cus(s);
  const bool wide = int8_gradient_tile(a.E, a.A, a.K, cus).cols == 256;
  a.ntn = (int32_t)ceil_div(a.K, (int64_t)(wide ? 256 : 128));
  const int64_t tiles = (ceil_div(a.A, (int64_t)kGradBM) + a.E - 1) * a.ntn;
  if (tiles > INT32_MAX) return NT_ERR_TOO_LARGE;
  const unsigned grid =
      (unsigned)std::min<int64_t>(tiles, (wide ? 2 : 3) * cus);
  auto go = [&](auto type) {
    typedef typename decltype(type)::type T;
    auto launch = [&](auto epilogue, auto input) {
      constexpr int EPI = decltype(epilogue)::value;
      constexpr bool IN = decltype(input)::value;
      if (wide)
        hipLaunchKernelGGL((int8_grad_kernel<T, EPI, 256, IN>), dim3(grid), dim3(kGradThreads), 0,
                           s, g);
      else
        hipLaunchKernelGGL((int8_grad_kernel<T, EPI, 128, IN>), dim3(grid), dim3(kGradThreads), 0,
                           s, g);
    };
    auto block = [&](auto input) {
      if (epi == kGradGelu) launch(std::integral_constant<int, kGradGelu>(), input);
      else launch(std::integral_constant<int, kGradSwiGLU>(), input);
    };
    if (epi == kGradTerms) return launch(std::integral_constant<int, kGradTerms>(), std::true_type());
    if (epi == kGradTermsDual)
      return launch(std::integral_constant<int, kGradTermsDual>(), std::true_type());
    if (in) return block(std::true_type());
    if constexpr (!std::is_same<T, float>::value) {
      if (epi == kGradPlain) launch(std::integral_constant<int, kGradPlain>(), std::false_type());
      else block(std::false_type());
    }
  };
  if (in && epi == kGradPlain) epi = kGradTerms;
  int8_by_type(dtype, go);
  return launch_status();
}

Int8Grad make_grad(const int8_t* w, const float* w_scales, const int32_t* offsets,
                   const void* dout, int64_t dout_pitch, int32_t E, int64_t A, int64_t K,
                   int64_t N, void* out) {
  Int8Grad g = {};
  g.rows.w = w, g.rows.w_scales = w_scales, g.rows.offsets = offsets;
  g.rows.E = E, g.rows.A = A, g.rows.K = K, g.rows.N = N, g.rows.out = out;
  g.dout = dout, g.pitch = dout_pitch;
  return g;
}

}  // namespace

// Half as wide where tiles of 256 columns (an expert's last one half full) are about as
// few as CUs: a step waits for its loads, and then twice as many run at a time (66
// tiles, 4,188 rows of terms, 2,048 to 512: 56 us for 80; 264, 512 to 2,048: 34 for 39;
// but 420, 871 rows, 4,096 to 14,336: 178 for 159, and 1,024 109 for 98).
Int8Tile int8_gradient_tile(int64_t E, int64_t A, int64_t K, int64_t cus) {
  const int64_t tiles = (ceil_div(A, (int64_t)kGradBM) + E / 2) * ceil_div(K, (int64_t)256);
  return {kGradBM, 4 * tiles > 5 * cus ? 256 : 128};
}

}  // namespace nt

using namespace nt;

extern "C" {

size_t nt_int8_terms_bytes(int dtype, int64_t A, int64_t N) {
  if (!int8_float(dtype) || A < 0 || A > kInt8MaxRows || N < 1 || N > kGradMaxN) return 0;
  return (size_t)((dtype == NT_F32 ? 3 : 2) * A * int8_pitch(N) * 2);
}

int nt_int8_rows_terms(int dtype, const void* dout, const int32_t* offsets, const float* w_scales,
                       int32_t E, int64_t A, int64_t N, void* terms, hipStream_t stream) {
  if (!int8_float(dtype)) return NT_ERR_DTYPE;
  if (E < 1 || A < 0 || N < 1) return NT_ERR_INVALID_ARG;
  if (E > NT_MAX_EXPERTS) return NT_ERR_TOO_MANY_EXPERTS;
  if (N > kGradMaxN || A > kInt8MaxRows) return NT_ERR_TOO_LARGE;
  if (A == 0) return NT_OK;
  if (dout == nullptr || w_scales == nullptr || terms == nullptr ||
      reinterpret_cast<uintptr_t>(terms) % 16 != 0 || (offsets == nullptr && E != 1))
    return NT_ERR_INVALID_ARG;
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    hipLaunchKernelGGL((int8_terms_kernel<T>), dim3((unsigned)ceil_div(A, (int64_t)kTermRows)),
                       dim3(kTermRows * kWave), 0, stream, dout, offsets, w_scales, E, A, N,
                       terms);
  });
  return launch_status();
}

int nt_int8_terms(const float* dout, const int32_t* offsets, const float* w_scales, int32_t E,
                  int64_t A, int64_t N, void* terms, hipStream_t stream) {
  return nt_int8_rows_terms(NT_F32, dout, offsets, w_scales, E, A, N, terms, stream);
}

int nt_int8_grouped_gemm_dx(int dtype, const int8_t* w, const float* w_scales,
                            const int32_t* offsets, const void* dout, int64_t dout_pitch,
                            int32_t E, int64_t A, int64_t K, int64_t N, void* dx,
                            hipStream_t stream) {
  return run_grad(dtype, kGradPlain,
                  make_grad(w, w_scales, offsets, dout, dout_pitch, E, A, K, N, dx), stream);
}

int nt_int8_grouped_gemm_dx_gelu(int dtype, const int8_t* w, const float* w_scales,
                                 const int32_t* offsets, const void* dout, int64_t dout_pitch,
                                 const float* act_grad, const float* up_scales, int32_t E,
                                 int64_t A, int64_t K, int64_t N, void* terms,
                                 hipStream_t stream) {
  Int8Grad g = make_grad(w, w_scales, offsets, dout, dout_pitch, E, A, K, N, terms);
  g.aux = act_grad, g.next = up_scales;
  return run_grad(dtype, kGradGelu, g, stream);
}

int nt_int8_grouped_gemm_dx_swiglu(int dtype, const int8_t* w, const float* w_scales,
                                   const int32_t* offsets, const void* dout, int64_t dout_pitch,
                                   const float* gate, const float* value,
                                   const float* gate_scales, const float* val_scales, int32_t E,
                                   int64_t A, int64_t K, int64_t N, void* gate_terms,
                                   void* val_terms, hipStream_t stream) {
  Int8Grad g = make_grad(w, w_scales, offsets, dout, dout_pitch, E, A, K, N, gate_terms);
  g.aux = gate, g.aux2 = value, g.next = gate_scales, g.next2 = val_scales;
  g.terms2 = val_terms;
  return run_grad(dtype, kGradSwiGLU, g, stream);
}

int nt_int8_grouped_gemm_dx_terms(int dtype, const int8_t* w, const int8_t* w2,
                                  const int32_t* offsets, const void* terms, const void* terms2,
                                  int32_t E, int64_t A, int64_t K, int64_t N, void* dx,
                                  hipStream_t stream) {
  Int8Grad g = make_grad(w, nullptr, offsets, terms, 0, E, A, K, N, dx);
  g.rows.w2 = w2, g.dout2 = terms2;
  if (w2 == nullptr && terms2 != nullptr) return NT_ERR_INVALID_ARG;
  return run_grad(dtype, w2 == nullptr ? kGradTerms : kGradTermsDual, g, stream);
}

}  // extern "C"
