// PyTorch-ROCm binding of the 8-bit integer experts and linear layers
// (nanotitan_int8.h): checks, outputs and workspaces, as torch_ext.cpp has them for
// the rest. Bringing activations to 8 bits and the products that follow are one
// call each, so that a layer's launches follow each other without Python between.
#include "nanotitan_int8.h"
#include "torch_common.hpp"

namespace {

using OptTensor = c10::optional<Tensor>;

void check_rows(const Tensor& x, const char* name) {
  check_device(x, name);
  TORCH_CHECK(x.dim() == 2 && x.size(1) >= 1 && x.is_contiguous(), name,
              " must be a contiguous [rows, columns]");
  const auto t = x.scalar_type();
  TORCH_CHECK(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, name,
              " must be float32, float16 or bfloat16");
}

// A weight of [E, K, N]: its integers in blocks and its scales.
struct Weight {
  const int8_t* codes;
  const float* scales;
  int32_t E;
  int64_t K, N;
};
Weight check_weight(const Tensor& codes, const Tensor& scales, int64_t K, const Tensor& like,
                    const char* name) {
  check_device(codes, name);
  check_same_device(like, {&codes, &scales});
  TORCH_CHECK(codes.scalar_type() == at::kChar && scales.scalar_type() == at::kFloat, name,
              " must be int8 integers with float32 scales");
  TORCH_CHECK(scales.dim() == 2 && scales.is_contiguous() && codes.is_contiguous(), name,
              " needs contiguous integers and scales [E, N]");
  const int64_t E = scales.size(0), N = scales.size(1);
  TORCH_CHECK(E >= 1 && N >= 1 && K >= 1 && E <= INT32_MAX, name, " must not be empty");
  const size_t bytes = nt_int8_weight_bytes((int32_t)E, K, N);
  TORCH_CHECK(bytes > 0, name, ": at most ", NT_MAX_EXPERTS, " experts, ", NT_INT8_MAX_K,
              " reduction rows and 2^22 columns, got [", E, ", ", K, ", ", N, "]");
  TORCH_CHECK((size_t)codes.numel() == bytes, name, " of [", E, ", ", K, ", ", N, "] must have ",
              bytes, " integers, has ", codes.numel());
  TORCH_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0, name,
              " must be 16-byte aligned");
  TORCH_CHECK(!scales.requires_grad(), name, " in 8 bits has no gradient: its scales need none");
  return {codes.data_ptr<int8_t>(), scales.data_ptr<float>(), (int32_t)E, K, N};
}

const int32_t* check_offsets(const OptTensor& offsets, const Tensor& x, int32_t E) {
  if (!offsets) {
    TORCH_CHECK(E == 1, "without expert_offset the weights must be of one expert, not ", E);
    return nullptr;
  }
  check_i32(*offsets, "expert_offset");
  check_same_device(x, {&*offsets});
  TORCH_CHECK(offsets->is_contiguous() && offsets->dim() == 1 && offsets->numel() == E + 1,
              "expert_offset must hold num_experts + 1 entries");
  return offsets->data_ptr<int32_t>();
}

// int8_rows(x) -> (codes [rows/16, f/64, 4, 16, 16], scales), and back.
std::tuple<Tensor, Tensor> int8_rows(Tensor x) {
  const OptTensor in = x;
  refuse_tangents({&in}, "int8_rows");
  check_rows(x, "x");
  c10::hip::HIPGuard guard(x.get_device());
  const int64_t rows = x.size(0), f = x.size(1);
  Tensor codes = at::empty({(rows + 15) / 16, nt_int8_pitch(f) / 64, 4, 16, 16},
                           x.options().dtype(at::kChar));
  Tensor scales = at::empty({rows}, x.options().dtype(at::kFloat));
  check_status(nt_int8_rows(dtype_code(x), x.data_ptr(), rows, f, codes.data_ptr<int8_t>(),
                            scales.data_ptr<float>(), stream_of(x)),
               "int8_rows");
  return {codes, scales};
}
Tensor int8_rows_decode(Tensor codes, Tensor scales, int64_t width, at::ScalarType dtype) {
  check_device(codes, "codes");
  check_f32(scales, "scales");
  check_same_device(codes, {&scales});
  TORCH_CHECK(codes.scalar_type() == at::kChar, "codes must be int8");
  TORCH_CHECK(width >= 1 && width <= NT_INT8_MAX_K && scales.dim() == 1 &&
                  scales.is_contiguous() && codes.is_contiguous() &&
                  codes.numel() == (scales.size(0) + 15) / 16 * 16 * nt_int8_pitch(width) &&
                  reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0,
              "expected contiguous codes [rows / 16, width / 64, 4, 16, 16], rounded up, and "
              "scales [rows] for width ", width);
  c10::hip::HIPGuard guard(codes.get_device());
  Tensor x = at::empty({scales.size(0), width}, codes.options().dtype(dtype));
  check_status(nt_int8_rows_decode(dtype_code(x), codes.data_ptr<int8_t>(),
                                   scales.data_ptr<float>(), scales.size(0), width, x.data_ptr(),
                                   stream_of(codes)),
               "int8_rows_decode");
  return x;
}

// int8_weight(W) -> (codes [E, N/64, K/64, 4, 4, 16, 16], scales [E, N]), and back.
std::tuple<Tensor, Tensor> int8_weight(Tensor W) {
  const OptTensor in = W;
  refuse_tangents({&in}, "int8_weight");
  check_device(W, "W");
  TORCH_CHECK(W.dim() == 3 && W.numel() > 0 && W.is_contiguous(),
              "W must be a contiguous [experts, in, out]");
  const auto t = W.scalar_type();
  TORCH_CHECK(t == at::kFloat || t == at::kHalf || t == at::kBFloat16,
              "W must be float32, float16 or bfloat16");
  const int64_t E = W.size(0), K = W.size(1), N = W.size(2);
  TORCH_CHECK(E <= NT_MAX_EXPERTS && nt_int8_weight_bytes((int32_t)E, K, N) > 0, "W: at most ",
              NT_MAX_EXPERTS, " experts, ", NT_INT8_MAX_K, " rows and 2^22 columns");
  c10::hip::HIPGuard guard(W.get_device());
  Tensor codes = at::empty({E, (N + 63) / 64, nt_int8_pitch(K) / 64, 4, 4, 16, 16},
                           W.options().dtype(at::kChar));
  Tensor scales = at::empty({E, N}, W.options().dtype(at::kFloat));
  Tensor ws = workspace(W, nt_int8_weight_workspace_bytes((int32_t)E, N));
  check_status(nt_int8_weight(dtype_code(W), W.data_ptr(), (int32_t)E, K, N,
                              codes.data_ptr<int8_t>(), scales.data_ptr<float>(), ws.data_ptr(),
                              ws.numel(), stream_of(W)),
               "int8_weight");
  return {codes, scales};
}
Tensor int8_weight_decode(Tensor codes, Tensor scales, int64_t K, at::ScalarType dtype) {
  const Weight w = check_weight(codes, scales, K, codes, "weight");
  c10::hip::HIPGuard guard(codes.get_device());
  Tensor W = at::empty({w.E, w.K, w.N}, codes.options().dtype(dtype));
  check_status(nt_int8_weight_decode(dtype_code(W), w.codes, w.scales, w.E, w.K, w.N,
                                     W.data_ptr(), stream_of(codes)),
               "int8_weight_decode");
  return W;
}

float* kept_or_null(const OptTensor& t) { return t ? t->data_ptr<float>() : nullptr; }

// x @ W, x's rows brought to 8 bits.
Tensor linear(const Tensor& x, const int32_t* off, const Weight& w) {
  const int64_t A = x.size(0);
  Tensor out = at::empty({A, w.N}, x.options());
  Tensor ws = workspace(x, nt_int8_linear_workspace_bytes(A, w.K));
  check_status(nt_int8_linear(dtype_code(x), x.data_ptr(), off, w.codes, w.scales, w.E, A, w.K,
                              w.N, out.data_ptr(), ws.data_ptr(), ws.numel(), stream_of(x)),
               "int8_linear");
  return out;
}

// int8_product(x, offsets, codes, scales) -> x @ W.
Tensor int8_product(Tensor x, OptTensor offsets, Tensor codes, Tensor scales) {
  const OptTensor in = x;
  refuse_tangents({&in}, "int8_grouped_gemm");
  check_rows(x, "X");
  const Weight w = check_weight(codes, scales, x.size(1), x, "weight");
  const int32_t* off = check_offsets(offsets, x, w.E);
  c10::hip::HIPGuard guard(x.get_device());
  return linear(x, off, w);
}

void check_down(const Weight& up, const Weight& down, int64_t d) {
  TORCH_CHECK(down.E == up.E && down.N == d, "expected down weights [", up.E, ", ", up.N, ", ", d,
              "], got [", down.E, ", ", down.K, ", ", down.N, "]");
}

// int8_swiglu_ffn(x, offsets, gate, value and out weights, keep) -> (y, gate, value).
std::tuple<Tensor, OptTensor, OptTensor> int8_swiglu_ffn(Tensor x, OptTensor offsets, Tensor wg,
                                                         Tensor sg, Tensor wv, Tensor sv,
                                                         Tensor wo, Tensor so, bool keep) {
  const OptTensor in = x;
  refuse_tangents({&in}, "int8_swiglu_ffn");
  check_rows(x, "X");
  const int64_t A = x.size(0), d = x.size(1);
  const Weight g = check_weight(wg, sg, d, x, "gate weight");
  const Weight v = check_weight(wv, sv, d, x, "value weight");
  TORCH_CHECK(v.E == g.E && v.N == g.N, "gate and value weights must be alike");
  const Weight o = check_weight(wo, so, g.N, x, "out weight");
  check_down(g, o, d);
  const int32_t* off = check_offsets(offsets, x, g.E);
  c10::hip::HIPGuard guard(x.get_device());
  Tensor hidden = at::empty({A, g.N}, x.options());
  OptTensor gate, value;
  if (keep) {
    gate = at::empty({A, g.N}, x.options().dtype(at::kFloat));
    value = at::empty_like(*gate);
  }
  {
    Tensor ws = workspace(x, nt_int8_linear_workspace_bytes(A, d));
    check_status(nt_int8_linear_swiglu(dtype_code(x), x.data_ptr(), off, g.codes, g.scales,
                                       v.codes, v.scales, g.E, A, d, g.N, hidden.data_ptr(),
                                       kept_or_null(gate), kept_or_null(value), ws.data_ptr(),
                                       ws.numel(), stream_of(x)),
                 "int8_linear_swiglu");
  }
  Tensor y = linear(hidden, off, o);
  return {y, gate, value};
}

// int8_gelu_ffn(x, offsets, up and down weights, keep) -> (y, gelu').
std::tuple<Tensor, OptTensor> int8_gelu_ffn(Tensor x, OptTensor offsets, Tensor wu, Tensor su,
                                            Tensor wd, Tensor sd, bool keep) {
  const OptTensor in = x;
  refuse_tangents({&in}, "int8_gelu_ffn");
  check_rows(x, "X");
  const int64_t A = x.size(0), d = x.size(1);
  const Weight u = check_weight(wu, su, d, x, "up weight");
  const Weight o = check_weight(wd, sd, u.N, x, "down weight");
  check_down(u, o, d);
  const int32_t* off = check_offsets(offsets, x, u.E);
  c10::hip::HIPGuard guard(x.get_device());
  Tensor act = at::empty({A, u.N}, x.options());
  OptTensor slope;
  if (keep) slope = at::empty({A, u.N}, x.options().dtype(at::kFloat));
  {
    Tensor ws = workspace(x, nt_int8_linear_workspace_bytes(A, d));
    check_status(nt_int8_linear_gelu(dtype_code(x), x.data_ptr(), off, u.codes, u.scales, u.E, A,
                                     d, u.N, act.data_ptr(), kept_or_null(slope), ws.data_ptr(),
                                     ws.numel(), stream_of(x)),
                 "int8_linear_gelu");
  }
  Tensor y = linear(act, off, o);
  return {y, slope};
}

Tensor new_terms(const Tensor& like, int64_t A, int64_t N) {
  return at::empty({like.scalar_type() == at::kFloat ? 3 : 2, A, nt_int8_pitch(N)},
                   like.options().dtype(at::kBFloat16));
}

// A gradient's rows for the products with the weights held: their terms (of float32
// always), or rows of 16-bit types of a multiple of 8 values, aligned.
struct GradIn {
  Weight w;
  const int32_t* off;
  int64_t A, pitch;
  Tensor rows;
};
GradIn check_dx(const Tensor& dout, const OptTensor& offsets, const Tensor& codes,
                const Tensor& scales, int64_t K, bool by_terms) {
  check_rows(dout, "dOut");
  const Weight w = check_weight(codes, scales, K, dout, "weight");
  const int32_t* off = check_offsets(offsets, dout, w.E);
  const int64_t A = dout.size(0), pitch = dout.size(1);
  if (by_terms || dout.scalar_type() == at::kFloat) {
    TORCH_CHECK(pitch == w.N, "dOut must have ", w.N, " columns, has ", pitch);
    c10::hip::HIPGuard guard(dout.get_device());
    Tensor terms = new_terms(dout, A, w.N);
    check_status(nt_int8_rows_terms(dtype_code(dout), dout.data_ptr(), off, w.scales, w.E, A, w.N,
                                    terms.data_ptr(), stream_of(dout)),
                 "int8_terms");
    return {w, off, A, 0, terms};
  }
  TORCH_CHECK(pitch == (w.N + 7) / 8 * 8 &&
                  reinterpret_cast<uintptr_t>(dout.data_ptr()) % 16 == 0,
              "dOut must be rows of ", w.N, " values, rounded up to a multiple of 8, 16-byte "
              "aligned");
  return {w, off, A, pitch, dout};
}
// What the forward kept [A, K], and the scales of the weights before [E, K].
void check_kept(const Tensor& t, int64_t rows, int64_t cols, const Tensor& like,
                const char* name) {
  check_f32(t, name);
  check_same_device(like, {&t});
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.is_contiguous(), name,
              " must be a contiguous [", rows, ", ", cols, "]");
}

// int8_dx(dOut, offsets, codes, scales, K, by_terms) -> dOut @ W^T.
Tensor int8_dx(Tensor dout, OptTensor offsets, Tensor codes, Tensor scales, int64_t K,
               bool by_terms) {
  const GradIn g = check_dx(dout, offsets, codes, scales, K, by_terms);
  c10::hip::HIPGuard guard(dout.get_device());
  Tensor dx = at::empty({g.A, K}, dout.options());
  check_status(nt_int8_grouped_gemm_dx(dtype_code(dout), g.w.codes, g.w.scales, g.off,
                                       g.rows.data_ptr(), g.pitch, g.w.E, g.A, K, g.w.N,
                                       dx.data_ptr(), stream_of(dout)),
               "int8_dx");
  return dx;
}
// The same and an activation's gradient, in terms for the up projections: (terms of
// up or gate, of value).
Tensor int8_dx_gelu(Tensor dout, Tensor slope, OptTensor offsets, Tensor codes, Tensor scales,
                    Tensor up_scales, int64_t K, bool by_terms) {
  const GradIn g = check_dx(dout, offsets, codes, scales, K, by_terms);
  check_kept(slope, g.A, K, dout, "gelu'");
  check_kept(up_scales, g.w.E, K, dout, "up scales");
  c10::hip::HIPGuard guard(dout.get_device());
  Tensor terms = new_terms(dout, g.A, K);
  check_status(nt_int8_grouped_gemm_dx_gelu(dtype_code(dout), g.w.codes, g.w.scales, g.off,
                                            g.rows.data_ptr(), g.pitch, slope.data_ptr<float>(),
                                            up_scales.data_ptr<float>(), g.w.E, g.A, K, g.w.N,
                                            terms.data_ptr(), stream_of(dout)),
               "int8_dx_gelu");
  return terms;
}
std::tuple<Tensor, Tensor> int8_dx_swiglu(Tensor dout, Tensor gate, Tensor value,
                                          OptTensor offsets, Tensor codes, Tensor scales,
                                          Tensor gate_scales, Tensor val_scales, int64_t K,
                                          bool by_terms) {
  const GradIn g = check_dx(dout, offsets, codes, scales, K, by_terms);
  check_kept(gate, g.A, K, dout, "gate");
  check_kept(value, g.A, K, dout, "value");
  check_kept(gate_scales, g.w.E, K, dout, "gate scales");
  check_kept(val_scales, g.w.E, K, dout, "value scales");
  c10::hip::HIPGuard guard(dout.get_device());
  Tensor tg = new_terms(dout, g.A, K), tv = new_terms(dout, g.A, K);
  check_status(nt_int8_grouped_gemm_dx_swiglu(
                   dtype_code(dout), g.w.codes, g.w.scales, g.off, g.rows.data_ptr(), g.pitch,
                   gate.data_ptr<float>(), value.data_ptr<float>(),
                   gate_scales.data_ptr<float>(), val_scales.data_ptr<float>(), g.w.E, g.A, K,
                   g.w.N, tg.data_ptr(), tv.data_ptr(), stream_of(dout)),
               "int8_dx_swiglu");
  return {tg, tv};
}
// int8_dx_terms(terms, second terms, offsets, codes, scales, second codes, K, dtype):
// their products with the weights that they hold the scales of.
Tensor int8_dx_terms(Tensor terms, OptTensor terms2, OptTensor offsets, Tensor codes,
                     Tensor scales, OptTensor codes2, int64_t K, at::ScalarType dtype) {
  check_device(terms, "terms");
  const Weight w = check_weight(codes, scales, K, terms, "weight");
  TORCH_CHECK(terms2.has_value() == codes2.has_value(), "each weight needs its terms");
  for (const Tensor* t : {&terms, terms2 ? &*terms2 : &terms}) {
    check_same_device(terms, {t});
    TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->is_contiguous() &&
                    t->dim() == 3 && t->size(0) == (dtype == at::kFloat ? 3 : 2) &&
                    t->size(1) == terms.size(1) && t->size(2) == nt_int8_pitch(w.N) &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "terms must be contiguous, aligned [2 or 3, rows, columns] of bfloat16");
  }
  if (codes2) check_weight(*codes2, scales, K, terms, "second weight");
  const int32_t* off = check_offsets(offsets, terms, w.E);
  c10::hip::HIPGuard guard(terms.get_device());
  Tensor dx = at::empty({terms.size(1), K}, terms.options().dtype(dtype));
  check_status(nt_int8_grouped_gemm_dx_terms(
                   dtype_code(dx), w.codes, codes2 ? codes2->data_ptr<int8_t>() : nullptr, off,
                   terms.data_ptr(), terms2 ? terms2->data_ptr() : nullptr, w.E, terms.size(1), K,
                   w.N, dx.data_ptr(), stream_of(terms)),
               "int8_dx_terms");
  return dx;
}

// int8_moe_few_tokens(x, up, value and down weights, top_k, router, logits) -> (out,
// gates, topk): moe_few_tokens on 8-bit weights.
std::tuple<Tensor, Tensor, Tensor> int8_moe_few_tokens(Tensor x, Tensor wu, Tensor su,
                                                       OptTensor wv, OptTensor sv, Tensor wd,
                                                       Tensor sd, int64_t top_k, OptTensor router,
                                                       OptTensor logits) {
  const OptTensor in = x;
  refuse_tangents({&in, &router, &logits}, "moe_few_tokens");
  check_rows(x, "x");
  const int64_t T = x.size(0), d = x.size(1);
  const Weight u = check_weight(wu, su, d, x, "up weight");
  const Weight o = check_weight(wd, sd, u.N, x, "down weight");
  check_down(u, o, d);
  TORCH_CHECK(wv.has_value() == sv.has_value(), "value weights need their scales");
  Weight v = {};
  if (wv) {
    v = check_weight(*wv, *sv, d, x, "value weight");
    TORCH_CHECK(v.E == u.E && v.N == u.N, "gate and value weights must be alike");
  }
  TORCH_CHECK(router.has_value() != logits.has_value(),
              "exactly one of the router's weight and logits is needed");
  const Tensor& r = router ? *router : *logits;
  check_f32(r, router ? "router weight" : "logits");
  check_same_device(x, {&r});
  TORCH_CHECK(r.is_contiguous() && r.dim() == 2 && r.size(0) == (router ? u.E : T) &&
                  r.size(1) == (router ? d : u.E),
              "expected a contiguous router weight [E,d] or logits [T,E]");
  TORCH_CHECK(T <= NT_FEW_TOKENS_MAX, "at most ", NT_FEW_TOKENS_MAX, " tokens, got ", T);
  TORCH_CHECK(top_k >= 1 && top_k <= u.E, "top_k must be in [1, num_experts]");
  c10::hip::HIPGuard guard(x.get_device());
  Tensor out = at::empty_like(x);
  Tensor gates = at::empty({T, top_k}, x.options().dtype(at::kFloat));
  Tensor topk = at::empty({T, top_k}, x.options().dtype(at::kInt));
  const int dt = dtype_code(x);
  Tensor ws = workspace(
      x, nt_int8_moe_few_tokens_workspace_bytes(dt, T, u.E, (int32_t)top_k, d, u.N));
  check_status(nt_int8_moe_few_tokens(dt, x.data_ptr(), f32_or_null(router), f32_or_null(logits),
                                      u.codes, u.scales, v.codes, v.scales, o.codes, o.scales, T,
                                      u.E, (int32_t)top_k, d, u.N, gates.data_ptr<float>(),
                                      topk.data_ptr<int32_t>(), out.data_ptr(), ws.data_ptr(),
                                      ws.numel(), stream_of(x)),
               "moe_few_tokens");
  return {out, gates, topk};
}

}  // namespace

void bind_int8(py::module& m) {
  m.def("int8_rows", &int8_rows, "Rows in 8-bit integers -> (codes, scales)");
  m.def("int8_rows_decode", &int8_rows_decode, "The rows that integers and scales hold");
  m.def("int8_weight", &int8_weight, "Weights in 8-bit integers -> (codes, scales)");
  m.def("int8_weight_decode", &int8_weight_decode, "The weights that integers and scales hold");
  m.def("int8_product", &int8_product, "Rows by 8-bit weights, grouped by expert");
  m.def("int8_swiglu_ffn", &int8_swiglu_ffn, "SwiGLU FFN on 8-bit weights -> (y, gate, value)");
  m.def("int8_gelu_ffn", &int8_gelu_ffn, "GELU FFN on 8-bit weights -> (y, gelu')");
  const auto by_terms = pybind11::arg("by_terms") = false;
  using a = pybind11::arg;
  m.def("int8_dx", &int8_dx, "Gradient rows by 8-bit weights, transposed", a("dout"), a("offsets"),
        a("codes"), a("scales"), a("K"), by_terms);
  m.def("int8_dx_gelu", &int8_dx_gelu, "Such a product times gelu' -> terms", a("dout"), a("slope"),
        a("offsets"), a("codes"), a("scales"), a("up_scales"), a("K"), by_terms);
  m.def("int8_dx_swiglu", &int8_dx_swiglu, "Such a product by SwiGLU's gradient -> (terms, terms)",
        a("dout"), a("gate"), a("value"), a("offsets"), a("codes"), a("scales"), a("gate_scales"),
        a("val_scales"), a("K"), by_terms);
  m.def("int8_dx_terms", &int8_dx_terms, "Terms by the integers of 8-bit weights, transposed");
  m.def("int8_moe_few_tokens", &int8_moe_few_tokens,
        "A whole MoE layer for few tokens on 8-bit weights -> (out, gates, topk)");
}
