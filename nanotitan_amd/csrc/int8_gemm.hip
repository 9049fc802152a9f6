// Expert-grouped products of 8-bit integers, with a scale for each row of the
// activations and each channel of the weights:
//
//   out[a, n] = (sum_k qx[a, k] qw[e, k, n]) sw[e, n] sx[a],   e the expert of row a
//
// Integer sums are exact, so an output does not depend on tiles or on the batch;
// int32 holds them up to 2^17 reduction rows. Two scalings and one rounding
// follow, or in float32 an activation: silu(gate) * value of two weight matrices
// side by side, or GELU.
//
// Many rows are bound by the matrix instructions (32,768 rows, 8 experts of 14,336 to
// 4,096: 1.70 to 1.82 ms, 2.1 to 2.3 Pop/s; the library's plain product of 16,384^3 reaches
// 2.35) and by what feeds them: a ring of three stages in LDS, filled directly, with
// operands that lie in memory as the instructions take them, and the next step's
// fragments read behind this one's instructions. Few rows are one read of the weights
// (int8_few.hip). In between an expert's last tile is part empty and its weights are
// read for few products (128 experts with 112 rows each, 2,048 to 768: 0.5 Pop/s).
#include <algorithm>

#include "gelu.hpp"
#include "gemm_common.hpp"
#include "int8.hpp"
#include "int8_gemm.hpp"

namespace nt {
namespace {

// ------------------------------------------------------------ tiled products

// One k-step is SB = 64 or 128 integers of each operand row. Operands are copied to
// LDS as they are, 1 KiB a load instruction: a lane's offset never changes, and what
// tells instructions and steps apart is uniform. Both go into the vector offset: the
// buffer's range does not cover a scalar one, and the last row block's and column
// group's tiles reach past the integers.

// The step's operands of `ROWS` rows (activations) or columns (weights): UNIT
// operands (one; a group's four) for each of its SB / 64 blocks, then the next 16
// rows (or 64 columns).
template <int ROWS, int UNIT, int SB, int NW>
struct OperandCopy {
  static constexpr int kBytes = ROWS * SB;
  static constexpr int kPer = kBytes / 1024 / NW;
  static_assert(kBytes / 1024 % NW == 0, "whole instructions for every wave");
  static constexpr int kGroup = UNIT * SB / 64;  // instructions of a row block
  i32x4_t rsrc;
  uint32_t lane_off;
  // From `base`, of which `bytes` are readable (what lies past them reads zeros).
  __device__ __forceinline__ void init(const int8_t* base, int64_t bytes, uint32_t off) {
    rsrc = make_rsrc(base, bytes);
    lane_off = off;
  }
  __device__ __forceinline__ void issue(int kt, uint32_t group, char* lds, int wave) const {
    const uint32_t l0 = lds_addr(lds);
    i32x4_t r;  // in scalar registers, wherever the tile loop keeps it
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_readfirstlane(rsrc[j]);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const uint32_t i = wave + u * NW;
      load16_to_lds(r, lane_off + __builtin_amdgcn_readfirstlane(
                                      i / kGroup * group + kt * (kGroup * 1024) +
                                      i % kGroup * 1024),
                    __builtin_amdgcn_readfirstlane(l0 + i * 1024u));
    }
  }
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Waits until only the last `younger` stages' loads (at most MOST count) are in
// flight: the counter's operand is a constant.
template <int MOST, int LOADS>
__device__ __forceinline__ void wait_stages(int younger) {
  if constexpr (MOST <= 0) {
    wait_vmcnt<0>();
  } else {
    if (younger >= MOST) wait_vmcnt<MOST * LOADS>();
    else wait_stages<MOST - 1, LOADS>(younger);
  }
}

// Where a wave's results lie. The weights' operand goes first, so lane l holds
// rows l % 16 of the row blocks, and of column group c and operand t columns 64 c +
// 16 (l / 16) + 4 t .. + 3.
template <typename T, int EPI, int AB, int CG>
__device__ __forceinline__ void int8_store(const i32x4 (&acc)[AB][EPI == kInt8SwiGLU ? 2 : 1][CG][4],
                                           const Int8Gemm& a, int64_t e, int64_t row0, int rows,
                                           int m0, int64_t n0, int lane) {
  typedef typename elem<T>::storage S;
  constexpr int MATS = EPI == kInt8SwiGLU ? 2 : 1;
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
      S o[16];
      float o2[16], o3[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        int8_epilogue<T, EPI>((float)acc[b][0][c][j / 4][j % 4] * sw[0][j] * sx,
                              MATS == 2 ? (float)acc[b][MATS - 1][c][j / 4][j % 4] *
                                              sw[MATS - 1][j] * sx
                                        : 0.f,
                              o[j], o2[j], o3[j]);
      const int64_t at = row * a.N + n;
      const int width = (int)(a.N - n < 16 ? a.N - n : 16);
      int8_put(static_cast<S*>(a.out) + at, width, o);
      if (EPI != kInt8Plain && a.out2 != nullptr) int8_put(a.out2 + at, width, o2);
      if (EPI == kInt8SwiGLU && a.out3 != nullptr) int8_put(a.out3 + at, width, o3);
    }
  }
}

template <typename T, int EPI, int BM, int BN, int WGM, int WGN, int NS>
__global__ void __launch_bounds__(WGM* WGN* kWave, BM* BN / (WGM * WGN) > 128 * 64 ? 1 : 2)
    int8_tile_kernel(Int8Gemm a) {
  constexpr int NW = WGM * WGN, SB = kInt8Block;
  constexpr int MATS = EPI == kInt8SwiGLU ? 2 : 1;
  constexpr int WM = BM / WGM, WN = BN / WGN / MATS;  // of each matrix
  constexpr int AB = WM / 16, CG = WN / 64;
  static_assert(WM % 16 == 0 && WN % 64 == 0, "whole operands");
  typedef OperandCopy<BM, 1, SB, NW> TA;
  typedef OperandCopy<BN / MATS, 4, SB, NW> TB;
  constexpr int kStage = TA::kBytes + MATS * TB::kBytes;
  __shared__ __attribute__((aligned(1024))) char smem[NS * kStage];
  __shared__ int32_t s_pref[NT_MAX_EXPERTS + 1];
  int8_row_tiles(a, BM, s_pref);
  const int64_t mtiles = __builtin_amdgcn_readfirstlane(s_pref[a.E]);
  // (more than that many only where offsets are malformed)
  const int64_t total = mtiles * a.ntn < INT32_MAX ? mtiles * a.ntn : INT32_MAX;
  // Tiles are dealt to the XCDs in contiguous ranges, as the 16-bit GEMMs' are.
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
  int64_t logical = t_beg + wg / kXcd;
  if (logical >= t_end) return;

  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WGN, wn = wave % WGN;
  const int64_t pitch = int8_pitch(a.K), groups = int8_groups(a.N);
  const int nk = (int)(pitch / SB);

  int e = 0, rows = 0;
  int64_t row0 = 0, col0 = 0;
  const uint32_t row_block = (uint32_t)(16 * pitch), group = (uint32_t)(kInt8Block * pitch);
  TA ta;
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
    // rows from any of 16 on: the lanes past the last of them go to the next 16
    const int64_t x0 = (row0 >> 4) * row_block;
    const uint32_t in16 = (uint32_t)(row0 & 15) + (lane & 15);
    ta.init(a.x + x0, int8_rows_bytes(a.A, pitch) - x0,
            (in16 >> 4) * row_block + (in16 & 15) * 16 + (lane >> 4) * 256);
#pragma unroll
    for (int i = 0; i < MATS; ++i) {
      const int64_t g0 = col0 / kInt8Block;
      tb[i].init((i == 0 ? a.w : a.w2) + (e * groups + g0) * group, (groups - g0) * group,
                 lane * 16);
    }
  };
  auto issue = [&](int kt, char* lds) {
    ta.issue(kt, row_block, lds, wave);
#pragma unroll
    for (int i = 0; i < MATS; ++i) tb[i].issue(kt, group, lds + TA::kBytes + i * TB::kBytes, wave);
  };
  constexpr int kLoads = TA::kPer + MATS * TB::kPer;

  // A k-step is multiplied from registers that the step before filled: after the
  // barrier of step kt every wave holds its operands of kt, so that stage's slot is
  // free for step kt + NS, and stage kt + 1 has landed and is read behind the
  // matrix instructions of kt.
  i32x4 acc[AB][MATS][CG][4];
  constexpr int kB = MATS * CG * 4;  // weight operands of a wave
  struct Operands {
    i32x4 x[AB], w[kB];
  };
  auto read = [&](const char* stage, Operands& o) {
#pragma unroll
    for (int b = 0; b < AB; ++b)
      o.x[b] = *reinterpret_cast<const i32x4*>(stage + (wm * AB + b) * 1024 + lane * 16);
#pragma unroll
    for (int j = 0; j < kB; ++j)
      o.w[j] = *reinterpret_cast<const i32x4*>(stage + TA::kBytes + j / (CG * 4) * TB::kBytes +
                                               (wn * CG + j / 4 % CG) * 4096 + j % 4 * 1024 +
                                               lane * 16);
  };
  auto multiply = [&](const Operands& o) {
#pragma unroll
    for (int b = 0; b < AB; ++b)
#pragma unroll
      for (int j = 0; j < kB; ++j) {
        i32x4& c = acc[b][j / (CG * 4)][j / 4 % CG][j % 4];
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(o.w[j], o.x[b], c, 0, 0, 0);
      }
  };
  // Every wave's reads are done and all loads but the `younger` last stages' have
  // landed (vector memory operations retire in order).
  auto arrive = [&](int younger) {
    wait_stages<NS - 2, kLoads>(younger);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  auto prefetch = [&]() {
#pragma unroll
    for (int s0 = 0; s0 < NS; ++s0)
      if (s0 < nk) issue(s0, smem + s0 * kStage);
  };
  setup(logical);
  prefetch();
  while (true) {
#pragma unroll
    for (int b = 0; b < AB; ++b)
#pragma unroll
      for (int i = 0; i < MATS; ++i)
#pragma unroll
        for (int c = 0; c < CG; ++c)
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[b][i][c][t] = i32x4{0, 0, 0, 0};
    Operands o0, o1;
    if (nk >= NS) wait_vmcnt<(NS - 1) * kLoads>();
    else wait_vmcnt<0>();
    asm volatile("s_barrier" ::: "memory");
    read(smem, o0);
    int slot = 0;
    auto step = [&](int kt, const Operands& now, Operands& then) {
      arrive(nk - 2 - kt);
      if (kt + NS < nk) issue(kt + NS, smem + slot * kStage);
      slot = slot + 1 == NS ? 0 : slot + 1;
      if (kt + 1 < nk) read(smem + slot * kStage, then);
      multiply(now);
    };
    for (int kt = 0; kt < nk; kt += 2) {  // (an even number: K is padded to 128)
      step(kt, o0, o1);
      step(kt + 1, o1, o0);
    }
    const int64_t next = logical + nbx;
    const int64_t se = e, srow = row0, scol = col0;
    const int srows = rows;
    const bool more = next < t_end;
    if (more) {  // no wave reads the stages any more
      setup(next);
      prefetch();
    }
    int8_store<T, EPI, AB, CG>(acc, a, se, srow, srows, wm * WM, scol + wn * WN, lane);
    if (!more) break;
    logical = next;
  }
}

template <typename T, int EPI, int BM, int BN, int WGM, int WGN, int NS>
int launch_tiles(Int8Gemm a, int per_cu, hipStream_t s) {
  constexpr int MATS = EPI == kInt8SwiGLU ? 2 : 1;
  a.ntn = (int32_t)ceil_div(a.N, (int64_t)(BN / MATS));
  const int64_t tiles = (ceil_div(a.A, (int64_t)BM) + a.E - 1) * a.ntn;  // at most
  if (tiles > INT32_MAX) return NT_ERR_TOO_LARGE;
  const int64_t grid = std::min<int64_t>(tiles, (int64_t)device_cus(s) * per_cu);
  hipLaunchKernelGGL((int8_tile_kernel<T, EPI, BM, BN, WGM, WGN, NS>), dim3((unsigned)grid),
                     dim3(WGM * WGN * kWave), 0, s, a);
  return launch_status();
}

// Which kernel. With few rows an expert the weights are read straight into registers
// (int8_few.hip), and where there are fewer 128x128 tiles than CUs and reading the
// weights once for every 64 rows takes less than a tile's k-steps: a step of 64 lasts
// 0.32 us whatever the tile holds, that reading runs at 4 TB/s (one expert, 14,336
// to 4,096: 64 rows 25 us against 72, 128 28 against 73; 4,096 to 14,336: 64 rows 18
// against 26, 128 29 against 27). Else tiles of 128x256 with two workgroups a CU: one's
// epilogue runs behind the other's products. Where these are less than about one
// and a half rounds of the chip's slots, tiles of half the width (E = 8, 4,000 rows
// of 4,096 to 4,096: 92 -> 79 us; 38,400 rows, E = 128, 2,048 to 768: 94 us against
// 99). Long reductions of many tiles take 256x256, which reads less from L2 and LDS
// for a product (32,768 rows, 14,336 to 4,096: 1,793 -> 1,692 us, 8,192: 990 -> 940,
// but 4,096: 442 -> 486; two matrices, 4,096 to 4,096: 969 -> 942 us, 2,048: 505 ->
// 512).
Int8Tile int8_tile(int epi, int64_t E, int64_t A, int64_t K, int64_t N, int64_t cus) {
  const bool two = epi == kInt8SwiGLU;
  const int64_t width = two ? 128 : 256;
  auto tiles = [&](int64_t rows) {  // expected: an expert's last tile is half full
    return (ceil_div(A, rows) + E / 2) * ceil_div(N, width);
  };
  const int64_t loads = ceil_div(A, 64) + E / 2;
  if (A <= 24 * E || ((ceil_div(A, 128) + E / 2) * ceil_div(N, two ? 64 : 128) <= cus &&
                      loads * N * (two ? 2 : 1) < 20000))
    return {0, 0};
  if (K >= (two ? 4096 : 8192) && tiles(256) >= 4 * cus) return {256, 256};
  if (tiles(128) >= 3 * cus) return {128, 256};
  return {128, 128};
}

template <typename T, int EPI>
int launch_by_size(const Int8Gemm& a, hipStream_t s) {
  constexpr int dtype = std::is_same<T, float>::value ? NT_F32
                        : std::is_same<T, f16>::value ? NT_F16 : NT_BF16;
  const Int8Tile tile = int8_tile(EPI, a.E, a.A, a.K, a.N, device_cus(s));
  if (tile.rows == 0) {
    launch_int8_stream(a, EPI, dtype, s);
    return launch_status();
  }
  if (tile.rows == 256) return launch_tiles<T, EPI, 256, 256, 4, 2, 3>(a, 1, s);
  if (tile.cols == 256) return launch_tiles<T, EPI, 128, 256, 2, 2, 3>(a, 2, s);
  if constexpr (EPI == kInt8SwiGLU) return launch_tiles<T, EPI, 128, 128, 4, 1, 3>(a, 2, s);
  else return launch_tiles<T, EPI, 128, 128, 2, 2, 3>(a, 3, s);
}

int check_int8(int dtype, const Int8Gemm& a) {
  if (!int8_float(dtype)) return NT_ERR_DTYPE;
  if (a.E < 1 || a.A < 0 || a.K < 1 || a.N < 1) return NT_ERR_INVALID_ARG;
  if (a.E > NT_MAX_EXPERTS) return NT_ERR_TOO_MANY_EXPERTS;
  if (a.K > kInt8MaxK || a.N > (1 << 22) || a.A > kInt8MaxRows) return NT_ERR_TOO_LARGE;
  return NT_OK;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int run_int8(int dtype, int epi, Int8Gemm a, hipStream_t s, void* ws = nullptr,
             size_t ws_bytes = 0) {
  const int st = check_int8(dtype, a);
  if (st != NT_OK || a.A == 0) return st;
  const bool two = epi == kInt8SwiGLU;
  if ((a.values == nullptr && (a.x == nullptr || a.x_scales == nullptr)) || a.w == nullptr ||
      a.w_scales == nullptr || a.out == nullptr || (two && (a.w2 == nullptr || a.w2_scales == nullptr)) ||
      (a.offsets == nullptr && a.E != 1) || (two && (a.out2 == nullptr) != (a.out3 == nullptr)) ||
      !aligned16(a.x) || !aligned16(a.w) || !aligned16(a.w2))
    return NT_ERR_INVALID_ARG;
  if (a.values != nullptr) {
    if (ws == nullptr || ws_bytes < nt_int8_linear_workspace_bytes(a.A, a.K) || !aligned16(ws))
      return NT_ERR_WORKSPACE;
    if (launch_int8_own(a, epi, dtype, s)) return launch_status();
    int8_t* codes = static_cast<int8_t*>(ws);
    float* scales = reinterpret_cast<float*>(codes + int8_rows_bytes(a.A, int8_pitch(a.K)));
    const int made = nt_int8_rows(dtype, a.values, a.A, a.K, codes, scales, s);
    if (made != NT_OK) return made;
    a.x = codes, a.x_scales = scales;
  }
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

int nt_int8_tile(int product, int32_t E, int64_t A, int64_t K, int64_t N, int32_t cus,
                 int32_t* rows, int32_t* columns) {
  if (product < NT_INT8_PLAIN || product > NT_INT8_GRADIENT || cus < 1 || rows == nullptr ||
      columns == nullptr)
    return NT_ERR_INVALID_ARG;
  Int8Gemm a = {};
  a.E = E, a.A = A, a.K = K, a.N = N;
  const int st = check_int8(NT_F32, a);
  if (st != NT_OK) return st;
  const Int8Tile tile = product == NT_INT8_GRADIENT ? int8_gradient_tile(E, A, K, cus)
                                                    : int8_tile(product, E, A, K, N, cus);
  *rows = tile.rows, *columns = tile.cols;
  return NT_OK;
}

size_t nt_int8_linear_workspace_bytes(int64_t A, int64_t K) {
  if (A < 0 || A > kInt8MaxRows || K < 1 || K > kInt8MaxK) return 0;
  return (size_t)(int8_rows_bytes(A, int8_pitch(K)) + round_up(A * 4, 16));
}

int nt_int8_linear(int dtype, const void* x, const int32_t* offsets, const int8_t* w,
                   const float* w_scales, int32_t E, int64_t A, int64_t K, int64_t N, void* out,
                   void* ws, size_t ws_bytes, hipStream_t stream) {
  Int8Gemm a = {};
  a.values = x, a.offsets = offsets, a.w = w, a.w_scales = w_scales;
  a.E = E, a.A = A, a.K = K, a.N = N, a.out = out;
  if (x == nullptr && A > 0) return NT_ERR_INVALID_ARG;
  return run_int8(dtype, kInt8Plain, a, stream, ws, ws_bytes);
}

int nt_int8_linear_swiglu(int dtype, const void* x, const int32_t* offsets, const int8_t* w_gate,
                          const float* gate_scales, const int8_t* w_val, const float* val_scales,
                          int32_t E, int64_t A, int64_t K, int64_t N, void* hidden, float* gate,
                          float* value, void* ws, size_t ws_bytes, hipStream_t stream) {
  Int8Gemm a = {};
  a.values = x, a.offsets = offsets, a.w = w_gate, a.w_scales = gate_scales;
  a.w2 = w_val, a.w2_scales = val_scales;
  a.E = E, a.A = A, a.K = K, a.N = N, a.out = hidden, a.out2 = gate, a.out3 = value;
  if (x == nullptr && A > 0) return NT_ERR_INVALID_ARG;
  return run_int8(dtype, kInt8SwiGLU, a, stream, ws, ws_bytes);
}

int nt_int8_linear_gelu(int dtype, const void* x, const int32_t* offsets, const int8_t* w,
                        const float* w_scales, int32_t E, int64_t A, int64_t K, int64_t N,
                        void* act, float* act_grad, void* ws, size_t ws_bytes,
                        hipStream_t stream) {
  Int8Gemm a = {};
  a.values = x, a.offsets = offsets, a.w = w, a.w_scales = w_scales;
  a.E = E, a.A = A, a.K = K, a.N = N, a.out = act, a.out2 = act_grad;
  if (x == nullptr && A > 0) return NT_ERR_INVALID_ARG;
  return run_int8(dtype, kInt8Gelu, a, stream, ws, ws_bytes);
}

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
                                int64_t N, void* hidden, float* gate, float* value,
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
                              float* act_grad, hipStream_t stream) {
  Int8Gemm a = {};
  a.x = x, a.x_scales = x_scales, a.offsets = offsets, a.w = w, a.w_scales = w_scales;
  a.E = E, a.A = A, a.K = K, a.N = N, a.out = act, a.out2 = act_grad;
  return run_int8(dtype, kInt8Gelu, a, stream);
}

}  // extern "C"
