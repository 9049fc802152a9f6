// Expert-grouped products of 8-bit integers, with a scale for each row of the
// activations and each channel of the weights:
//
//   out[a, n] = (sum_k qx[a, k] qw[e, k, n]) sw[e, n] sx[a],   e the expert of row a
//
// Integer sums are exact, so an output does not depend on tiles or on the batch;
// int32 holds them up to 2^17 reduction rows. Two scalings and one rounding
// follow, or in float32 an activation: silu(gate) * value of two weight matrices
// side by side, or GELU.
#include <algorithm>

#include "gelu.hpp"
#include "gemm_common.hpp"
#include "int8.hpp"
#include "int8_gemm.hpp"

namespace nt {
namespace {

// ------------------------------------------------------------ tiled products

// One k-step is 128 integers of each operand row. The activations' tile lies in
// LDS as the 16-bit GEMMs' K-major tiles do (64 two-byte elements a row: the loads
// and the bank swizzle do not know what the bytes are); the weights' blocks are
// copied as they are.
constexpr int kStepBytes = 128;
constexpr int kStepBlocks = kStepBytes / kInt8Block;

// Copies of weight blocks to LDS: BN / 64 column groups x 2 blocks of 4 KiB, 1 KiB
// an instruction.
template <int BN, int NW>
struct WeightTile {
  static constexpr int kBytes = BN * kStepBytes;
  static constexpr int kPer = kBytes / 1024 / NW;
  static_assert(kBytes / 1024 % NW == 0, "whole instructions for every wave");
  i32x4_t rsrc;
  uint32_t group;  // bytes from one column group to the next
  // Of expert e's matrix (column groups from g0 on); groups past the last read zeros.
  __device__ __forceinline__ void init(const int8_t* matrix, int64_t g0, int64_t groups,
                                       int64_t pitch) {
    rsrc = make_rsrc(matrix + g0 * pitch * kInt8Block, (groups - g0) * pitch * kInt8Block);
    group = (uint32_t)(pitch * kInt8Block);
  }
  __device__ __forceinline__ void issue(int64_t kt, char* lds, int wave, int lane) const {
    const uint32_t l0 = lds_addr(lds);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = wave + u * NW;  // instruction: group i / 8, KiB i % 8 of the step's two blocks
      const uint32_t at = (uint32_t)(i / 8) * group + (uint32_t)kt * (kStepBytes * kInt8Block) +
                          (uint32_t)(i % 8) * 1024u;
      load16_to_lds(rsrc, (uint32_t)lane * 16u + at,
                    __builtin_amdgcn_readfirstlane(l0 + (uint32_t)i * 1024u));
    }
  }
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Where a wave's results lie. The weights' operand goes first, so lane l holds
// rows l % 16 of the row blocks, and of column group c and operand t columns 64 c +
// 16 (l / 16) + 4 t .. + 3.
template <typename T, int EPI, int AB, int CG>
__device__ __forceinline__ void int8_store(const i32x4 (&acc)[AB][EPI == kInt8SwiGLU ? 2 : 1][CG][4],
                                           const Int8Gemm& a, int64_t e, int64_t row0, int rows,
                                           int m0, int64_t n0, int lane) {
  typedef typename elem<T>::storage S;
  constexpr int MATS = EPI == kInt8SwiGLU ? 2 : 1;
  const bool whole = a.N % 16 == 0 && a.wide_stores;
#pragma unroll
  for (int c = 0; c < CG; ++c) {
    const int64_t n = n0 + 64 * c + 16 * (lane >> 4);
    float sw[MATS][16];
#pragma unroll
    for (int i = 0; i < MATS; ++i) {
      const float* s = (i == 0 ? a.w_scales : a.w2_scales) + e * a.N;
#pragma unroll
      for (int j = 0; j < 16; ++j) sw[i][j] = n + j < a.N ? s[n + j] : 0.f;
    }
#pragma unroll
    for (int b = 0; b < AB; ++b) {
      const int m = m0 + 16 * b + (lane & 15);
      if (m >= rows || n >= a.N) continue;
      const int64_t row = row0 + m;
      const float sx = a.x_scales[row];
      S o[3][16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        int8_epilogue<T, EPI>((float)acc[b][0][c][j / 4][j % 4] * sw[0][j] * sx,
                              MATS == 2 ? (float)acc[b][MATS - 1][c][j / 4][j % 4] *
                                              sw[MATS - 1][j] * sx
                                        : 0.f,
                              o[0][j], o[1][j], o[2][j]);
      int8_put<T, EPI>(a, row * a.N + n, (int)(a.N - n < 16 ? a.N - n : 16), whole, o);
    }
  }
}

template <typename T, int EPI, int BM, int BN, int WGM, int WGN, int NS>
__global__ void __launch_bounds__(WGM* WGN* kWave, 2)
    int8_tile_kernel(Int8Gemm a) {
  constexpr int NW = WGM * WGN;
  constexpr int MATS = EPI == kInt8SwiGLU ? 2 : 1;
  constexpr int WM = BM / WGM, WN = BN / WGN / MATS;  // of each matrix
  constexpr int AB = WM / 16, CG = WN / 64;
  static_assert(WM % 16 == 0 && WN % 64 == 0, "whole operands");
  typedef OperandTile<BM, true, 64, NW> TA;
  typedef WeightTile<BN / MATS, NW> TB;
  constexpr int kStage = TA::kBytes + MATS * TB::kBytes;
  __shared__ __attribute__((aligned(1024))) char smem[NS * kStage];
  __shared__ int32_t s_pref[NT_MAX_EXPERTS + 1];
  int8_row_tiles(a, BM, s_pref);
  const int64_t mtiles = s_pref[a.E];
  const int64_t total = mtiles * a.ntn;
  // Tiles are dealt to the XCDs in contiguous ranges, as the 16-bit GEMMs' are.
  constexpr int kXcd = 8;
  const int64_t G = gridDim.x, wg = blockIdx.x;
  const int xcd = (int)(wg % kXcd);
  const int64_t q = G / kXcd, r = G % kXcd;
  const int64_t before = xcd * q + (xcd < r ? xcd : r);
  const int64_t nbx = q + (xcd < r ? 1 : 0);
  const int64_t t_end = xcd_range_start(total, before + nbx, G, s_pref, a.E, a.ntn);
  const int64_t t_beg = xcd_range_start(total, before, G, s_pref, a.E, a.ntn);
  int64_t logical = t_beg + wg / kXcd;
  if (logical >= t_end) return;

  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WGN, wn = wave % WGN;
  FragReader<BM, true, AB, 64> fa;
  fa.init(wm * WM, lane);
  const int64_t pitch = int8_pitch(a.K), groups = int8_groups(a.N);
  const int nk = (int)(pitch / kStepBytes);

  int e = 0, rows = 0;
  int64_t row0 = 0, col0 = 0;
  const int8_t* xa = nullptr;
  TA ta;
  ta.init(pitch / 2, wave, lane);
  TB tb[MATS];
  auto setup = [&](int64_t t) {
    int64_t r0, r1, mtl;
    int nt;
    expert_tile_coords(t, s_pref, a.E, a.ntn, e, mtl, nt);
    int8_expert_rows(a, e, r0, r1);
    e = __builtin_amdgcn_readfirstlane(e);
    nt = __builtin_amdgcn_readfirstlane(nt);
    row0 = (int64_t)__builtin_amdgcn_readfirstlane((int)(r0 + mtl * BM));
    const int64_t left = (int64_t)__builtin_amdgcn_readfirstlane((int)r1) - row0;
    rows = (int)(left < BM ? left : BM);
    col0 = (int64_t)nt * (BN / MATS);
    xa = a.x + row0 * pitch;
#pragma unroll
    for (int i = 0; i < MATS; ++i)
      tb[i].init((i == 0 ? a.w : a.w2) + e * groups * kInt8Block * pitch, col0 / kInt8Block, groups,
                 pitch);
  };
  auto issue = [&](int kt, char* lds) {
    ta.issue(xa + (int64_t)kt * kStepBytes, (rows - 1) * pitch + kStepBytes, lds, 64, wave);
#pragma unroll
    for (int i = 0; i < MATS; ++i) tb[i].issue(kt, lds + TA::kBytes + i * TB::kBytes, wave, lane);
  };
  constexpr int kLoads = TA::kPer + MATS * TB::kPer;
  setup(logical);
#pragma unroll
  for (int s0 = 0; s0 < NS - 1; ++s0)
    if (s0 < nk) issue(s0, smem + s0 * kStage);

  i32x4 acc[AB][MATS][CG][4];
  constexpr int kB = MATS * CG * 4;  // weight operands of a wave and substep
  auto compute = [&](const char* sa) {
    const char* sb = sa + TA::kBytes;
    auto read_b = [&](int j, int ks) {
      const int i = j / (CG * 4), c = j / 4 % CG, t = j % 4;
      return *reinterpret_cast<const i32x4*>(sb + i * TB::kBytes +
                                             ((wn * CG + c) * 2 + ks) * 4096 + t * 1024 +
                                             lane * 16);
    };
    auto read_a = [&](int b, int ks) { return fa.template read<i32x4>(sa, b, ks); };
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      // the operand with fewer blocks is held, the other streams
      if constexpr (kB <= AB) {
        i32x4 held[kB];
#pragma unroll
        for (int j = 0; j < kB; ++j) held[j] = read_b(j, ks);
#pragma unroll
        for (int b = 0; b < AB; ++b) {
          const i32x4 x = read_a(b, ks);
#pragma unroll
          for (int j = 0; j < kB; ++j) {
            i32x4& o = acc[b][j / (CG * 4)][j / 4 % CG][j % 4];
            o = __builtin_amdgcn_mfma_i32_16x16x64_i8(held[j], x, o, 0, 0, 0);
          }
        }
      } else {
        i32x4 held[AB];
#pragma unroll
        for (int b = 0; b < AB; ++b) held[b] = read_a(b, ks);
#pragma unroll
        for (int j = 0; j < kB; ++j) {
          const i32x4 w = read_b(j, ks);
#pragma unroll
          for (int b = 0; b < AB; ++b) {
            i32x4& o = acc[b][j / (CG * 4)][j / 4 % CG][j % 4];
            o = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, held[b], o, 0, 0, 0);
          }
        }
      }
    }
  };

  while (true) {
#pragma unroll
    for (int b = 0; b < AB; ++b)
#pragma unroll
      for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int c = 0; c < CG; ++c)
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[b][i][c][t] = i32x4{0, 0, 0, 0};
    int slot = 0;
    for (int kt = 0; kt < nk; ++kt) {
      // This stage has landed when at most the younger stages' loads are in flight.
      if (nk - 1 - kt >= NS - 2) wait_vmcnt<(NS - 2) * kLoads>();
      else wait_vmcnt<0>();
      __syncthreads();
      if (kt + NS - 1 < nk) {
        int fill = slot + NS - 1;
        if (fill >= NS) fill -= NS;
        issue(kt + NS - 1, smem + fill * kStage);
      }
      compute(smem + slot * kStage);
      slot = slot + 1 == NS ? 0 : slot + 1;
    }
    __syncthreads();  // every wave is done with the stages
    const int64_t next = logical + nbx;
    const int64_t se = e, srow = row0, scol = col0;
    const int srows = rows;
    const bool more = next < t_end;
    if (more) {
      setup(next);
#pragma unroll
      for (int s0 = 0; s0 < NS - 1; ++s0)
        if (s0 < nk) issue(s0, smem + s0 * kStage);
    }
    int8_store<T, EPI, AB, CG>(acc, a, se, srow, srows, wm * WM, scol + wn * WN, lane);
    if (!more) break;
    logical = next;
  }
}

template <typename T, int EPI, int BM, int BN, int WGM, int WGN, int NS>
void launch_tiles(Int8Gemm a, int per_cu, hipStream_t s) {
  constexpr int MATS = EPI == kInt8SwiGLU ? 2 : 1;
  a.ntn = (int32_t)ceil_div(a.N, (int64_t)(BN / MATS));
  const int64_t tiles = (ceil_div(a.A, (int64_t)BM) + a.E - 1) * a.ntn;  // at most
  const int64_t grid = std::min<int64_t>(tiles, (int64_t)device_cus(s) * per_cu);
  hipLaunchKernelGGL((int8_tile_kernel<T, EPI, BM, BN, WGM, WGN, NS>), dim3((unsigned)grid),
                     dim3(WGM * WGN * kWave), 0, s, a);
}

template <typename T, int EPI>
int launch_by_size(const Int8Gemm& a, hipStream_t s) {
  const int64_t mean = ceil_div(a.A, (int64_t)a.E);
  constexpr int dtype = std::is_same<T, float>::value ? NT_F32
                        : std::is_same<T, f16>::value ? NT_F16 : NT_BF16;
  if (mean <= 64) {
    launch_int8_stream(a, EPI, dtype, s);
  } else if constexpr (EPI == kInt8SwiGLU) {
    if (mean <= 256) launch_tiles<T, EPI, 128, 128, 4, 1, 2>(a, 2, s);
    else launch_tiles<T, EPI, 256, 256, 4, 2, 2>(a, 1, s);
  } else {
    if (mean <= 256) launch_tiles<T, EPI, 128, 128, 2, 2, 2>(a, 2, s);
    else launch_tiles<T, EPI, 256, 256, 2, 4, 2>(a, 1, s);
  }
  return launch_status();
}

int check_int8(int dtype, const Int8Gemm& a) {
  if (!int8_float(dtype)) return NT_ERR_DTYPE;
  if (a.E < 1 || a.A < 0 || a.K < 1 || a.N < 1) return NT_ERR_INVALID_ARG;
  if (a.E > NT_MAX_EXPERTS) return NT_ERR_TOO_MANY_EXPERTS;
  if (a.K > kInt8MaxK || a.N > (1 << 22) || a.A > INT32_MAX - 512) return NT_ERR_TOO_LARGE;
  return NT_OK;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int run_int8(int dtype, int epi, Int8Gemm a, hipStream_t s) {
  const int st = check_int8(dtype, a);
  if (st != NT_OK || a.A == 0) return st;
  const bool two = epi == kInt8SwiGLU;
  if (a.x == nullptr || a.x_scales == nullptr || a.w == nullptr || a.w_scales == nullptr ||
      a.out == nullptr || (two && (a.w2 == nullptr || a.w2_scales == nullptr)) ||
      (a.offsets == nullptr && a.E != 1) || (two && (a.out2 == nullptr) != (a.out3 == nullptr)) ||
      !aligned16(a.x) || !aligned16(a.w) || !aligned16(a.w2))
    return NT_ERR_INVALID_ARG;
  a.wide_stores = aligned16(a.out) && aligned16(a.out2) && aligned16(a.out3);
  int result = NT_OK;
  int8_by_type(dtype, [&](auto type) {
    typedef typename decltype(type)::type T;
    result = epi == kInt8Plain    ? launch_by_size<T, kInt8Plain>(a, s)
             : epi == kInt8SwiGLU ? launch_by_size<T, kInt8SwiGLU>(a, s)
                                  : launch_by_size<T, kInt8Gelu>(a, s);
  });
  return result;
}

}  // namespace
}  // namespace nt

using namespace nt;

extern "C" {

int nt_int8_grouped_gemm(int dtype, const int8_t* x, const float* x_scales,
                         const int32_t* offsets, const int8_t* w, const float* w_scales,
                         int32_t E, int64_t A, int64_t K, int64_t N, void* out,
                         hipStream_t stream) {
  Int8Gemm a = {};
  a.x = x, a.x_scales = x_scales, a.offsets = offsets, a.w = w, a.w_scales = w_scales;
  a.E = E, a.A = A, a.K = K, a.N = N, a.out = out;
  return run_int8(dtype, kInt8Plain, a, stream);
}

int nt_int8_grouped_gemm_swiglu(int dtype, const int8_t* x, const float* x_scales,
                                const int32_t* offsets, const int8_t* w_gate,
                                const float* gate_scales, const int8_t* w_val,
                                const float* val_scales, int32_t E, int64_t A, int64_t K,
                                int64_t N, void* hidden, void* gate, void* value,
                                hipStream_t stream) {
  Int8Gemm a = {};
  a.x = x, a.x_scales = x_scales, a.offsets = offsets, a.w = w_gate, a.w_scales = gate_scales;
  a.w2 = w_val, a.w2_scales = val_scales;
  a.E = E, a.A = A, a.K = K, a.N = N, a.out = hidden, a.out2 = gate, a.out3 = value;
  return run_int8(dtype, kInt8SwiGLU, a, stream);
}

int nt_int8_grouped_gemm_gelu(int dtype, const int8_t* x, const float* x_scales,
                              const int32_t* offsets, const int8_t* w, const float* w_scales,
                              int32_t E, int64_t A, int64_t K, int64_t N, void* act,
                              void* act_grad, hipStream_t stream) {
  Int8Gemm a = {};
  a.x = x, a.x_scales = x_scales, a.offsets = offsets, a.w = w, a.w_scales = w_scales;
  a.E = E, a.A = A, a.K = K, a.N = N, a.out = act, a.out2 = act_grad;
  return run_int8(dtype, kInt8Gelu, a, stream);
}

}  // extern "C"
