/*
 * nanotitan_int8.h — C ABI of the 8-bit integer experts and linear layers on the
 * MI355X (gfx950): part of libnanotitan_moe.so, with the element type and status
 * codes, the calling rules and nt_strerror() of nanotitan_moe.h.
 *
 * Weights are held as integers with a float32 scale for each expert and output
 * channel, activations as integers with a scale for each row:
 *   s = max(max|v| / 127, 2^-126),  q = the integer nearest to v / s, ties to even.
 * A row or channel with an infinity or a NaN has a NaN scale and zero integers.
 * Products are exact int32 sums, scaled in float32 and rounded once. Sums run over
 * at most NT_INT8_MAX_K values, calls over at most NT_INT8_MAX_ROWS rows. Integers given by a caller are -127..127.
 *
 * Integers lie as the operands of the matrix instructions. Rows [A, f], 16 rows of
 * nt_int8_pitch(f) (a multiple of 128, zeros past f) after another,
 * nt_int8_rows_bytes(A, f) in all:
 *   codes[a / 16][k / 64][g][a % 16][k % 16],  g = k % 64 / 16.
 * Weights, nt_int8_weight_bytes(E, K, N) in all:
 *   codes[e][n / 64][k / 64][t][g][i][k % 16],  n % 64 = 16 (i / 4) + 4 t + i % 4,
 * n padded with zeros to a multiple of 64, k to one of 128; scales are [E, N].
 * Integers are 16-byte aligned. Activations are f32, f16 or bf16.
 * No counterpart in the reference, whose experts keep their training type
 * (src/model/feed_fwd.py:39-122).
 */
#ifndef NANOTITAN_INT8_H
#define NANOTITAN_INT8_H

#include "nanotitan_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NT_INT8_MAX_K (1 << 17)
#define NT_INT8_MAX_ROWS ((1 << 24) - 1)

int64_t nt_int8_pitch(int64_t f);
size_t nt_int8_rows_bytes(int64_t rows, int64_t f);
size_t nt_int8_weight_bytes(int32_t E, int64_t K, int64_t N);

/* Rows x [rows, f] to codes and scales [rows], and the values q s that they hold in
 * dtype (rounded once; past the type's largest: that). */
int nt_int8_rows(int dtype, const void* x, int64_t rows, int64_t f, int8_t* codes, float* scales,
                 hipStream_t stream);
int nt_int8_rows_decode(int dtype, const int8_t* codes, const float* scales, int64_t rows,
                        int64_t f, void* x, hipStream_t stream);

/* Weights W [E, K, N] to codes and scales, and back. The workspace (4-byte aligned)
 * holds the channels' maxima. */
size_t nt_int8_weight_workspace_bytes(int32_t E, int64_t N);
int nt_int8_weight(int dtype, const void* W, int32_t E, int64_t K, int64_t N, int8_t* codes,
                   float* scales, void* ws, size_t ws_bytes, hipStream_t stream);
int nt_int8_weight_decode(int dtype, const int8_t* codes, const float* scales, int32_t E,
                          int64_t K, int64_t N, void* W, hipStream_t stream);

/* out[a,:] = x[a] @ W[e] for the rows a of expert e: x as codes and scales of A rows
 * (nt_int8_rows), offsets as nt_grouped_gemm takes them, or NULL with E = 1 (a linear
 * layer of all rows). Rows >= offsets[E] are not written. out [A, N] of dtype. */
int nt_int8_grouped_gemm(int dtype, const int8_t* x, const float* x_scales,
                         const int32_t* offsets, const int8_t* w, const float* w_scales,
                         int32_t E, int64_t A, int64_t K, int64_t N, void* out,
                         hipStream_t stream);

/* Both projections of a gated block, its activation and the product:
 * hidden = silu(x @ W_gate[e]) * (x @ W_val[e]) in float32, rounded once. gate and
 * value [A, N] in float32 are what a backward needs (both NULL: not written). */
int nt_int8_grouped_gemm_swiglu(int dtype, const int8_t* x, const float* x_scales,
                                const int32_t* offsets, const int8_t* w_gate,
                                const float* gate_scales, const int8_t* w_val,
                                const float* val_scales, int32_t E, int64_t A, int64_t K,
                                int64_t N, void* hidden, float* gate, float* value,
                                hipStream_t stream);

/* act = gelu(x @ W[e]) (erf), and gelu' of the same in float32 (NULL: not written). */
int nt_int8_grouped_gemm_gelu(int dtype, const int8_t* x, const float* x_scales,
                              const int32_t* offsets, const int8_t* w, const float* w_scales,
                              int32_t E, int64_t A, int64_t K, int64_t N, void* act,
                              float* act_grad, hipStream_t stream);

/* How the products of these sizes are tiled on a chip of `cus` CUs, by the expected tiles
 * of evenly spread experts: rows and columns (of SwiGLU both matrices' together) of a tile,
 * or 0 and 0 where the weights are streamed. Of NT_INT8_GRADIENT K are the columns. No
 * result depends on it. */
enum { NT_INT8_PLAIN = 0, NT_INT8_SWIGLU = 1, NT_INT8_GELU = 2, NT_INT8_GRADIENT = 3 };
int nt_int8_tile(int product, int32_t E, int64_t A, int64_t K, int64_t N, int32_t cus,
                 int32_t* rows, int32_t* columns);

/* The same three from rows x [A, K] of dtype, which they bring to 8 bits themselves:
 * the bits of nt_int8_rows and the product. The workspace (16-byte aligned, contents
 * arbitrary) is written before it is read: calls that cannot overlap may share one. */
size_t nt_int8_linear_workspace_bytes(int64_t A, int64_t K);
int nt_int8_linear(int dtype, const void* x, const int32_t* offsets, const int8_t* w,
                   const float* w_scales, int32_t E, int64_t A, int64_t K, int64_t N, void* out,
                   void* ws, size_t ws_bytes, hipStream_t stream);
int nt_int8_linear_swiglu(int dtype, const void* x, const int32_t* offsets, const int8_t* w_gate,
                          const float* gate_scales, const int8_t* w_val, const float* val_scales,
                          int32_t E, int64_t A, int64_t K, int64_t N, void* hidden, float* gate,
                          float* value, void* ws, size_t ws_bytes, hipStream_t stream);
int nt_int8_linear_gelu(int dtype, const void* x, const int32_t* offsets, const int8_t* w,
                        const float* w_scales, int32_t E, int64_t A, int64_t K, int64_t N,
                        void* act, float* act_grad, void* ws, size_t ws_bytes,
                        hipStream_t stream);

/* Gradients through frozen 8-bit weights; the rounding of x to 8 bits is passed
 * straight through. dx = dout @ W[e]^T [A, K]: sums in float32, one rounding.
 * f16 and bf16: the weights are the values held, rounded to dtype. Row r of dout is at
 * r * dout_pitch, a multiple of 8 from N on; columns from N to the next multiple of 8
 * are read and must be finite. dout is 16-byte aligned.
 * f32, and f16 and bf16 with dout_pitch 0: dout stands for its terms (below) with the
 * weights' scales, which meet the integers themselves, so no weight is rounded; w_scales is
 * not read then, nor dout_pitch of f32. */
int nt_int8_grouped_gemm_dx(int dtype, const int8_t* w, const float* w_scales,
                            const int32_t* offsets, const void* dout, int64_t dout_pitch,
                            int32_t E, int64_t A, int64_t K, int64_t N, void* dx,
                            hipStream_t stream);

/* Terms: a gradient [A, N] times the scales [E, N] of the weights that it will meet, as
 * sums of bfloat16 numbers: two, to 2^-17, where gradients are f16 or bf16, three, to
 * 2^-25, where they are f32 (a product with a scale below 2^-100: to fewer bits).
 * [terms][A][nt_int8_pitch(N)], 16-byte aligned, columns from N on zero to the next
 * multiple of 16 (the rest is not written, nor read).
 * nt_int8_terms_bytes is their size (0: too large). nt_int8_rows_terms makes them of rows
 * dout [A, N] of dtype, nt_int8_terms of float32 ones. */
size_t nt_int8_terms_bytes(int dtype, int64_t A, int64_t N);
int nt_int8_rows_terms(int dtype, const void* dout, const int32_t* offsets, const float* w_scales,
                       int32_t E, int64_t A, int64_t N, void* terms, hipStream_t stream);
int nt_int8_terms(const float* dout, const int32_t* offsets, const float* w_scales, int32_t E,
                  int64_t A, int64_t N, void* terms, hipStream_t stream);

/* The gradient through a feed-forward block, in two products. The first takes dout, as
 * above, to the gradient of the up projections, that times the float32 act_grad
 * (dx_gelu), or by SwiGLU's from gate and value as the forward kept them (dx_swiglu),
 * where w is the down projection [E, K, N]. It is not rounded to dtype: what is written
 * are its terms for up projections of the scales given [E, K]. The second takes terms
 * times the up projections' integers (w2 and terms2 NULL: of one) to dx [A, K], rounded
 * once to dtype; N is the terms' width. */
int nt_int8_grouped_gemm_dx_gelu(int dtype, const int8_t* w, const float* w_scales,
                                 const int32_t* offsets, const void* dout, int64_t dout_pitch,
                                 const float* act_grad, const float* up_scales, int32_t E,
                                 int64_t A, int64_t K, int64_t N, void* terms,
                                 hipStream_t stream);
int nt_int8_grouped_gemm_dx_swiglu(int dtype, const int8_t* w, const float* w_scales,
                                   const int32_t* offsets, const void* dout, int64_t dout_pitch,
                                   const float* gate, const float* value,
                                   const float* gate_scales, const float* val_scales, int32_t E,
                                   int64_t A, int64_t K, int64_t N, void* gate_terms,
                                   void* val_terms, hipStream_t stream);
int nt_int8_grouped_gemm_dx_terms(int dtype, const int8_t* w, const int8_t* w2,
                                  const int32_t* offsets, const void* terms, const void* terms2,
                                  int32_t E, int64_t A, int64_t K, int64_t N, void* dx,
                                  hipStream_t stream);

/* nt_moe_few_tokens on 8-bit weights (w_val NULL: GELU): tokens and hidden values go
 * to 8 bits row by row, the hidden ones from their values in dtype. Everything else,
 * the limits of sizes and the workspace's rules are nt_moe_few_tokens'; d, f <=
 * NT_INT8_MAX_K. */
size_t nt_int8_moe_few_tokens_workspace_bytes(int dtype, int64_t T, int32_t E, int32_t k,
                                              int64_t d, int64_t f);
int nt_int8_moe_few_tokens(int dtype, const void* x, const float* router, const float* logits,
                           const int8_t* w_up, const float* up_scales, const int8_t* w_val,
                           const float* val_scales, const int8_t* w_down,
                           const float* down_scales, int64_t T, int32_t E, int32_t k, int64_t d,
                           int64_t f, float* gates, int32_t* topk, void* out, void* ws,
                           size_t ws_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* NANOTITAN_INT8_H */
