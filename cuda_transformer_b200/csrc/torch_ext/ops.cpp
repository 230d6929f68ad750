// ops.cpp -- torch.ops.cuda_transformer.* registrations over the C ABI.
//
// Keeps the reference's operator library name and every schema string
// verbatim (Transformer_launchers/bindings.cpp:3, linear_layer.cu:101-102,
// softmax_layer.cu:83-84, gelu_activation.cu:80-81, flash_attn_launcher.cu:145-146,
// causal_self_attn_layer.cu:135-136) so cuda_transformer/ops.py, the autograd
// functions and gpt/gpt.py bind unchanged.  Like the reference launchers this
// shim owns allocation: outputs are dense torch tensors on the input's device
// and scratch comes from the caching allocator.  Unlike them it guards the
// device, checks dtypes, and maps C-ABI status codes to RuntimeError.
//
// Precision of the tensor-core kernels: CUDA_TRANSFORMER_PRECISION =
// "3xtf32" (default, FP32-accurate), "tf32" or "fp32" (CUDA cores); the *_ex
// operators take it explicitly (0 = 3xtf32, 1 = tf32, 2 = fp32).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <cstdlib>
#include <cstring>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "ct_b200.h"

namespace cuda_transformer {
namespace {

using at::Tensor;

int default_precision() {
  static const int p = [] {
    const char* e = std::getenv("CUDA_TRANSFORMER_PRECISION");
    if (!e || !*e) return (int)CT_PRECISION_3XTF32;
    std::string s(e);
    if (s == "3xtf32" || s == "fp32acc") return (int)CT_PRECISION_3XTF32;
    if (s == "tf32") return (int)CT_PRECISION_TF32;
    if (s == "fp32" || s == "simt") return (int)CT_PRECISION_FP32;
    TORCH_CHECK(false, "CUDA_TRANSFORMER_PRECISION must be 3xtf32, tf32 or fp32, got ", s);
  }();
  return p;
}

void check_rc(int rc, const char* op) {
  TORCH_CHECK(rc == CT_OK, op, ": ", ct_status_string(rc));
}

void check_cuda_f32(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be float32");
}

void* cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Attention operands must be addressable by TMA (unit stride along head_dim,
// 16-byte aligned base and strides); anything else is copied once.
Tensor tma_ready(const Tensor& t) {
  bool ok = t.stride(3) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) == 0;
  for (int i = 0; i < 3 && ok; ++i) ok = (t.stride(i) % 4) == 0;
  return ok ? t : t.contiguous();
}

void strides4(const Tensor& t, int64_t out[4]) {
  for (int i = 0; i < 4; ++i) out[i] = t.stride(i);
}

// ------------------------------------------------------------ FlashAttention
std::tuple<Tensor, Tensor> fa2_fwd_impl(const Tensor& Q0, const Tensor& K0, const Tensor& V0,
                                        bool causal, int64_t precision) {
  check_cuda_f32(Q0, "Q");
  check_cuda_f32(K0, "K");
  check_cuda_f32(V0, "V");
  TORCH_CHECK(Q0.dim() == 4 && K0.sizes() == Q0.sizes() && V0.sizes() == Q0.sizes(),
              "Q, K, V must be [B, nh, T, hs] of equal shape");
  c10::cuda::CUDAGuard guard(Q0.device());
  const Tensor Q = tma_ready(Q0), K = tma_ready(K0), V = tma_ready(V0);
  const int64_t B = Q.size(0), H = Q.size(1), T = Q.size(2), D = Q.size(3);
  auto opt = Q.options();
  Tensor O = at::empty({B, H, T, D}, opt);
  Tensor L = at::empty({B, H, T}, opt);
  int64_t qs[4], ks[4], vs[4];
  strides4(Q, qs);
  strides4(K, ks);
  strides4(V, vs);
  check_rc(ct_fa2_fwd(Q.data_ptr<float>(), qs, K.data_ptr<float>(), ks, V.data_ptr<float>(), vs,
                      O.data_ptr<float>(), L.data_ptr<float>(), B, H, T, D, causal ? 1 : 0,
                      (int)precision, cur_stream()),
           "flash_attention_fwd");
  return {O, L};
}

std::tuple<Tensor, Tensor, Tensor> fa2_bwd_impl(const Tensor& Q0, const Tensor& K0,
                                                const Tensor& V0, const Tensor& O0,
                                                const Tensor& dO0, const Tensor& L, bool causal,
                                                int64_t precision) {
  check_cuda_f32(Q0, "Q");
  check_cuda_f32(K0, "K");
  check_cuda_f32(V0, "V");
  check_cuda_f32(O0, "O");
  check_cuda_f32(dO0, "dO");
  check_cuda_f32(L, "L");
  TORCH_CHECK(Q0.dim() == 4 && K0.sizes() == Q0.sizes() && V0.sizes() == Q0.sizes() &&
                  O0.sizes() == Q0.sizes() && dO0.sizes() == Q0.sizes(),
              "Q, K, V, O, dO must be [B, nh, T, hs] of equal shape");
  TORCH_CHECK(L.dim() == 3 && L.size(0) == Q0.size(0) && L.size(1) == Q0.size(1) &&
                  L.size(2) == Q0.size(2),
              "L must be [B, nh, T]");
  c10::cuda::CUDAGuard guard(Q0.device());
  const Tensor Q = tma_ready(Q0), K = tma_ready(K0), V = tma_ready(V0), O = O0,
               dO = tma_ready(dO0);
  const int64_t B = Q.size(0), H = Q.size(1), T = Q.size(2), D = Q.size(3);
  auto opt = Q.options();
  Tensor dQ = at::empty({B, H, T, D}, opt);
  Tensor dK = at::empty({B, H, T, D}, opt);
  Tensor dV = at::empty({B, H, T, D}, opt);
  const size_t ws_bytes = ct_fa2_bwd_workspace_size(B, H, T, D);
  Tensor ws = at::empty({(int64_t)std::max<size_t>(ws_bytes, 16)}, opt.dtype(at::kByte));
  int64_t qs[4], ks[4], vs[4], os[4], gs[4], ls[3] = {L.stride(0), L.stride(1), L.stride(2)};
  strides4(Q, qs);
  strides4(K, ks);
  strides4(V, vs);
  strides4(O, os);
  strides4(dO, gs);
  check_rc(ct_fa2_bwd(Q.data_ptr<float>(), qs, K.data_ptr<float>(), ks, V.data_ptr<float>(), vs,
                      O.data_ptr<float>(), os, dO.data_ptr<float>(), gs, L.data_ptr<float>(), ls,
                      dQ.data_ptr<float>(), dK.data_ptr<float>(), dV.data_ptr<float>(),
                      ws.data_ptr(), ws_bytes, B, H, T, D, causal ? 1 : 0, (int)precision,
                      cur_stream()),
           "flash_attention_bwd");
  return {dQ, dK, dV};
}

std::tuple<Tensor, Tensor> flash_attention_fwd(Tensor Q, Tensor K, Tensor V, bool causal) {
  return fa2_fwd_impl(Q, K, V, causal, default_precision());
}
std::tuple<Tensor, Tensor, Tensor> flash_attention_bwd(Tensor Q, Tensor K, Tensor V, Tensor O,
                                                       Tensor dO, Tensor L, bool causal) {
  return fa2_bwd_impl(Q, K, V, O, dO, L, causal, default_precision());
}
std::tuple<Tensor, Tensor> flash_attention_fwd_ex(Tensor Q, Tensor K, Tensor V, bool causal,
                                                  int64_t precision) {
  return fa2_fwd_impl(Q, K, V, causal, precision);
}
std::tuple<Tensor, Tensor, Tensor> flash_attention_bwd_ex(Tensor Q, Tensor K, Tensor V, Tensor O,
                                                          Tensor dO, Tensor L, bool causal,
                                                          int64_t precision) {
  return fa2_bwd_impl(Q, K, V, O, dO, L, causal, precision);
}

// ----------------------------------------------------------------- Linear
// x: (batch, m, k); weights: (k, n) or (1 | batch, k, n) "pre-transposed";
// bias: (n,); out: (batch, m, n)  -- linear_layer.cu:24-70.
// A [b, r, c] operand of the tensor-core linear layer must have a unit stride
// in one of its last two dimensions, the other strides 16-byte multiples (or
// extent 1) and a 16-byte aligned base (TMA).  Otherwise it is copied into a
// layout with unit last stride and rows padded to 4 floats, viewed back at its
// logical size (the kernel never reads the padding: TMA zero-fills past the
// logical extent).  Vocabulary-sized outputs (n = 65) and their gradients need
// this; the FP32 CUDA-core path takes any strides.
Tensor linear_operand(const Tensor& t) {
  auto al = [](int64_t stride, int64_t extent) { return extent <= 1 || (stride % 4) == 0; };
  const bool base = (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) == 0;
  const bool batch_ok = al(t.stride(0), t.size(0));
  const bool kmaj = t.stride(2) == 1 && al(t.stride(1), t.size(1));
  const bool mnmaj = t.stride(1) == 1 && al(t.stride(2), t.size(2));
  if (base && batch_ok && (kmaj || mnmaj)) return t;
  const int64_t cpad = (t.size(2) + 3) / 4 * 4;
  Tensor buf = at::empty({t.size(0), t.size(1), cpad}, t.options());
  Tensor view = buf.narrow(2, 0, t.size(2));
  view.copy_(t);
  return view;
}

Tensor fma_impl(const Tensor& x0, Tensor weights0, const Tensor& bias, int64_t precision) {
  if (weights0.dim() == 2) weights0 = weights0.unsqueeze(0);
  TORCH_CHECK(x0.dim() == 3, "x must be a 3D tensor (batch, m, k)");
  check_cuda_f32(x0, "x");
  check_cuda_f32(weights0, "weights");
  c10::cuda::CUDAGuard guard0(x0.device());
  const bool tc = precision != (int64_t)CT_PRECISION_FP32;
  const Tensor x = tc && x0.numel() > 0 ? linear_operand(x0) : x0;
  Tensor weights = tc && weights0.numel() > 0 ? linear_operand(weights0) : weights0;
  const int64_t batch = x.size(0), m = x.size(1), k = x.size(2), n = weights.size(2);
  TORCH_CHECK(weights.size(1) == k, "weights.size(1) must match x.size(2)");
  TORCH_CHECK(bias.size(0) == n, "bias.size(0) must match weights.size(2)");
  check_cuda_f32(bias, "bias");
  TORCH_CHECK(weights.size(0) == 1 || weights.size(0) == batch,
              "weights batch must be 1 or match x");
  Tensor out = at::empty({batch, m, n}, x.options());
  const int64_t xs[3] = {x.stride(0), x.stride(1), x.stride(2)};
  const int64_t wsd[3] = {weights.stride(0), weights.stride(1), weights.stride(2)};
  // per-tile counters of the split-K schedule (a few hundred bytes)
  const size_t wsb = ct_linear_workspace_size(batch, m, k, n);
  Tensor ws = at::empty({(int64_t)std::max<size_t>(wsb, 16)}, x.options().dtype(at::kByte));
  check_rc(ct_linear_fwd_ws(x.data_ptr<float>(), xs, weights.data_ptr<float>(), wsd,
                            bias.data_ptr<float>(), bias.stride(0), out.data_ptr<float>(), batch,
                            m, k, n, weights.size(0), (int)precision, ws.data_ptr(), wsb,
                            cur_stream()),
           "cuda_fma");
  return out;
}

Tensor cuda_fma(Tensor x, Tensor weights, Tensor bias) {
  return fma_impl(x, weights, bias, default_precision());
}
Tensor cuda_fma_ex(Tensor x, Tensor weights, Tensor bias, int64_t precision) {
  return fma_impl(x, weights, bias, precision);
}

// The linear layer with its neighbours fused in (ct_linear_fwd_ex): epilogue
// 0 none, 1 GELU (returns out = x W + b and act = gelu(out)), 2 GELU gradient
// (out = (x W + b) * gelu'(act_in)); want_colsum also returns the column sums
// of `weights` over its reduction index (db when weights is dY; batch 1).
// Returns (out, act or an empty tensor, colsum or an empty tensor).
std::tuple<Tensor, Tensor, Tensor> linear_fused(Tensor x0, Tensor weights0, Tensor bias,
                                                int64_t precision, int64_t epilogue,
                                                std::optional<Tensor> act_in0, bool want_colsum) {
  if (weights0.dim() == 2) weights0 = weights0.unsqueeze(0);
  TORCH_CHECK(x0.dim() == 3, "x must be a 3D tensor (batch, m, k)");
  check_cuda_f32(x0, "x");
  check_cuda_f32(weights0, "weights");
  check_cuda_f32(bias, "bias");
  c10::cuda::CUDAGuard guard0(x0.device());
  const bool tc = precision != (int64_t)CT_PRECISION_FP32;
  const Tensor x = tc && x0.numel() > 0 ? linear_operand(x0) : x0;
  const Tensor weights = tc && weights0.numel() > 0 ? linear_operand(weights0) : weights0;
  const int64_t batch = x.size(0), m = x.size(1), k = x.size(2), n = weights.size(2);
  TORCH_CHECK(weights.size(1) == k, "weights.size(1) must match x.size(2)");
  TORCH_CHECK(bias.size(0) == n, "bias.size(0) must match weights.size(2)");
  TORCH_CHECK(weights.size(0) == 1 || weights.size(0) == batch, "weights batch must be 1 or match x");
  TORCH_CHECK(!want_colsum || batch == 1, "column sums need batch 1");
  Tensor out = at::empty({batch, m, n}, x.options());
  Tensor act = epilogue == CT_EPILOGUE_GELU ? at::empty({batch, m, n}, x.options())
                                            : at::empty({0}, x.options());
  Tensor cs = want_colsum ? at::empty({n}, x.options()) : at::empty({0}, x.options());
  Tensor act_in;
  if (epilogue == CT_EPILOGUE_GELU_GRAD) {
    TORCH_CHECK(act_in0.has_value(), "the GELU-gradient epilogue needs act_in");
    act_in = act_in0->contiguous();
    check_cuda_f32(act_in, "act_in");
    TORCH_CHECK(act_in.numel() == batch * m * n, "act_in must have batch*m*n elements");
  }
  const int64_t xs[3] = {x.stride(0), x.stride(1), x.stride(2)};
  const int64_t wsd[3] = {weights.stride(0), weights.stride(1), weights.stride(2)};
  const size_t wsb = ct_linear_workspace_size(batch, m, k, n);
  Tensor ws = at::empty({(int64_t)std::max<size_t>(wsb, 16)}, x.options().dtype(at::kByte));
  check_rc(ct_linear_fwd_ex(x.data_ptr<float>(), xs, weights.data_ptr<float>(), wsd,
                            bias.data_ptr<float>(), bias.stride(0), out.data_ptr<float>(), batch, m,
                            k, n, weights.size(0), (int)precision, (int)epilogue,
                            epilogue == CT_EPILOGUE_GELU ? act.data_ptr<float>() : nullptr,
                            epilogue == CT_EPILOGUE_GELU_GRAD ? act_in.data_ptr<float>() : nullptr,
                            want_colsum ? cs.data_ptr<float>() : nullptr, 0, ws.data_ptr(), wsb,
                            cur_stream()),
           "linear_fused");
  return {out, act, cs};
}

// out += x W + bias (and colsum += column sums of weights, when given); out
// dense (batch, m, n).
void linear_accumulate_(Tensor out, std::optional<Tensor> colsum, Tensor x0, Tensor weights0,
                        Tensor bias, int64_t precision) {
  if (weights0.dim() == 2) weights0 = weights0.unsqueeze(0);
  TORCH_CHECK(x0.dim() == 3, "x must be a 3D tensor (batch, m, k)");
  check_cuda_f32(x0, "x");
  check_cuda_f32(weights0, "weights");
  check_cuda_f32(bias, "bias");
  check_cuda_f32(out, "out");
  c10::cuda::CUDAGuard guard0(x0.device());
  const bool tc = precision != (int64_t)CT_PRECISION_FP32;
  const Tensor x = tc && x0.numel() > 0 ? linear_operand(x0) : x0;
  const Tensor weights = tc && weights0.numel() > 0 ? linear_operand(weights0) : weights0;
  const int64_t batch = x.size(0), m = x.size(1), k = x.size(2), n = weights.size(2);
  TORCH_CHECK(weights.size(1) == k && bias.size(0) == n, "linear_accumulate_: shape mismatch");
  TORCH_CHECK(out.is_contiguous() && out.numel() == batch * m * n, "out must be dense (batch, m, n)");
  float* csp = nullptr;
  if (colsum.has_value()) {
    check_cuda_f32(*colsum, "colsum");
    TORCH_CHECK(colsum->is_contiguous() && colsum->numel() == n && batch == 1,
                "colsum must be a dense (n,) tensor, batch 1");
    csp = colsum->data_ptr<float>();
  }
  const int64_t xs[3] = {x.stride(0), x.stride(1), x.stride(2)};
  const int64_t wsd[3] = {weights.stride(0), weights.stride(1), weights.stride(2)};
  const size_t wsb = ct_linear_workspace_size(batch, m, k, n);
  Tensor ws = at::empty({(int64_t)std::max<size_t>(wsb, 16)}, x.options().dtype(at::kByte));
  check_rc(ct_linear_fwd_ex(x.data_ptr<float>(), xs, weights.data_ptr<float>(), wsd,
                            bias.data_ptr<float>(), bias.stride(0), out.data_ptr<float>(), batch, m,
                            k, n, weights.size(0), (int)precision, CT_EPILOGUE_NONE, nullptr,
                            nullptr, csp, 1, ws.data_ptr(), wsb, cur_stream()),
           "linear_accumulate_");
}

// ------------------------------------------------------------ cross entropy
// loss per row; logits (rows, vocab), row stride free, overwritten with
// softmax - onehot(targets).  targets int64 (rows,).
Tensor cross_entropy_fwd_bwd_(Tensor logits, Tensor targets, int64_t ignore_index) {
  check_cuda_f32(logits, "logits");
  TORCH_CHECK(logits.dim() == 2 && logits.stride(1) == 1, "logits must be (rows, vocab), unit column stride");
  TORCH_CHECK(targets.is_cuda() && targets.scalar_type() == at::kLong, "targets must be int64 on the GPU");
  TORCH_CHECK(targets.numel() == logits.size(0), "one target per row");
  c10::cuda::CUDAGuard guard(logits.device());
  const Tensor t = targets.contiguous();
  Tensor loss = at::empty({logits.size(0)}, logits.options());
  check_rc(ct_cross_entropy_fwd_bwd(logits.data_ptr<float>(), logits.stride(0), logits.size(0),
                                    logits.size(1), t.data_ptr<int64_t>(), ignore_index,
                                    loss.data_ptr<float>(), cur_stream()),
           "cross_entropy_fwd_bwd_");
  return loss;
}

// dy: (batch, m, n) -> db: (n,)  -- linear_layer.cu:72-97.
Tensor db_calculation(Tensor dy) {
  check_cuda_f32(dy, "dy");
  TORCH_CHECK(dy.dim() == 3, "dy must be a 3D tensor");
  c10::cuda::CUDAGuard guard(dy.device());
  const int64_t batch = dy.size(0), m = dy.size(1), n = dy.size(2);
  Tensor db = at::empty({n}, dy.options());
  const size_t wsb = ct_bias_grad_workspace_size(batch, m, n);
  Tensor ws = at::empty({(int64_t)std::max<size_t>(wsb, 16)}, dy.options().dtype(at::kByte));
  const int64_t s[3] = {dy.stride(0), dy.stride(1), dy.stride(2)};
  check_rc(ct_bias_grad(dy.data_ptr<float>(), s, db.data_ptr<float>(), batch, m, n, ws.data_ptr(),
                        wsb, cur_stream()),
           "db_calculation");
  return db;
}

// ---------------------------------------------------------------- Softmax
Tensor cuda_softmax(Tensor x) {
  TORCH_CHECK(x.dim() == 3, "x must be a 3D tensor");
  check_cuda_f32(x, "x");
  TORCH_CHECK(x.is_contiguous(), "x must be contiguous");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor out = at::empty_like(x);
  const int64_t n = x.size(2);
  check_rc(ct_softmax_fwd(x.data_ptr<float>(), out.data_ptr<float>(), x.size(0) * x.size(1), n,
                          cur_stream()),
           "cuda_softmax");
  return out;
}

Tensor cuda_softmax_bwd(Tensor probs, Tensor dp) {
  TORCH_CHECK(probs.dim() == 3, "probs must be a 3D tensor");
  check_cuda_f32(probs, "probs");
  TORCH_CHECK(probs.is_contiguous(), "probs must be contiguous");
  TORCH_CHECK(dp.dim() == 3, "dp must be a 3D tensor");
  check_cuda_f32(dp, "dp");
  TORCH_CHECK(dp.is_contiguous(), "dp must be contiguous");
  TORCH_CHECK(dp.sizes() == probs.sizes(), "dp must match probs");
  c10::cuda::CUDAGuard guard(probs.device());
  Tensor out = at::empty_like(probs);
  check_rc(ct_softmax_bwd(probs.data_ptr<float>(), dp.data_ptr<float>(), out.data_ptr<float>(),
                          probs.size(0) * probs.size(1), probs.size(2), cur_stream()),
           "cuda_softmax_bwd");
  return out;
}

// ------------------------------------------------------------------- GELU
Tensor gelu_activation(Tensor x) {
  check_cuda_f32(x, "x");
  TORCH_CHECK(x.is_contiguous(), "x must be contiguous");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor out = at::empty_like(x);
  check_rc(ct_gelu_fwd(x.data_ptr<float>(), out.data_ptr<float>(), x.numel(), cur_stream()),
           "gelu_activation");
  return out;
}

Tensor gelu_activation_bwd(Tensor x, Tensor dy) {
  check_cuda_f32(x, "x");
  TORCH_CHECK(x.is_contiguous(), "x must be contiguous");
  check_cuda_f32(dy, "dy");
  TORCH_CHECK(dy.is_contiguous(), "dy must be contiguous");
  TORCH_CHECK(dy.numel() == x.numel(), "dy must match x");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor out = at::empty_like(x);
  check_rc(ct_gelu_bwd(x.data_ptr<float>(), dy.data_ptr<float>(), out.data_ptr<float>(),
                       x.numel(), cur_stream()),
           "gelu_activation_bwd");
  return out;
}

// -------------------------------------------------------------- LayerNorm
// New surface (the reference's LayerNorm is a torch module, gpt/gpt.py:47-59).
std::tuple<Tensor, Tensor, Tensor> layernorm_fwd(Tensor x, Tensor gamma, Tensor beta, double eps) {
  check_cuda_f32(x, "x");
  check_cuda_f32(gamma, "gamma");
  check_cuda_f32(beta, "beta");
  TORCH_CHECK(x.is_contiguous() && gamma.is_contiguous() && beta.is_contiguous(),
              "layernorm inputs must be contiguous");
  const int64_t n = x.size(-1);
  TORCH_CHECK(gamma.numel() == n && beta.numel() == n, "gamma/beta must have x.size(-1) elements");
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = n ? x.numel() / n : 0;
  Tensor y = at::empty_like(x);
  Tensor mean = at::empty({rows}, x.options());
  Tensor rstd = at::empty({rows}, x.options());
  check_rc(ct_layernorm_fwd(x.data_ptr<float>(), gamma.data_ptr<float>(), beta.data_ptr<float>(),
                            y.data_ptr<float>(), mean.data_ptr<float>(), rstd.data_ptr<float>(),
                            rows, n, (float)eps, cur_stream()),
           "layernorm_fwd");
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layernorm_bwd(Tensor x, Tensor gamma, Tensor mean, Tensor rstd,
                                                 Tensor dy0) {
  check_cuda_f32(x, "x");
  check_cuda_f32(gamma, "gamma");
  check_cuda_f32(mean, "mean");
  check_cuda_f32(rstd, "rstd");
  check_cuda_f32(dy0, "dy");
  TORCH_CHECK(x.is_contiguous() && gamma.is_contiguous(), "layernorm inputs must be contiguous");
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor dy = dy0.contiguous();
  const int64_t n = x.size(-1), rows = n ? x.numel() / n : 0;
  Tensor dx = at::empty_like(x);
  Tensor dg = at::empty({n}, x.options());
  Tensor db = at::empty({n}, x.options());
  const size_t wsb = ct_layernorm_bwd_workspace_size(rows, n);
  Tensor ws = at::empty({(int64_t)std::max<size_t>(wsb, 16)}, x.options().dtype(at::kByte));
  check_rc(ct_layernorm_bwd(x.data_ptr<float>(), gamma.data_ptr<float>(), mean.data_ptr<float>(),
                            rstd.data_ptr<float>(), dy.data_ptr<float>(), dx.data_ptr<float>(),
                            dg.data_ptr<float>(), db.data_ptr<float>(), rows, n, ws.data_ptr(),
                            wsb, cur_stream()),
           "layernorm_bwd");
  return {dx, dg, db};
}

// ---------------------------------------------------------- token generation
// A dense CUDA tensor beside `of`, allocated without a trip through the
// dispatcher (which costs as much as a kernel's launch).
Tensor empty_like_of(at::IntArrayRef sizes, at::ScalarType type, const Tensor& of) {
  return at::detail::empty_cuda(sizes, type, of.device(), std::nullopt);
}

int dtype_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return CT_DTYPE_F32;
    case at::kBFloat16: return CT_DTYPE_BF16;
    case at::kHalf: return CT_DTYPE_F16;
    default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16");
  }
}

void check_on(const Tensor& t, const Tensor& first, at::ScalarType type, const char* name) {
  TORCH_CHECK(t.device() == first.device(), name, " must be on ", first.device());
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type);
}

// A dense 1-D operand of n elements (copied once if it is not dense); a null
// pointer when it is absent.
template <class T>
const T* vector_of(const std::optional<Tensor>& t, int64_t n, const Tensor& first,
                   at::ScalarType type, const char* name, Tensor* keep) {
  if (!t.has_value()) return nullptr;
  check_on(*t, first, type, name);
  TORCH_CHECK(t->dim() == 1 && t->size(0) == n, name, " must have ", n, " elements");
  *keep = t->contiguous();
  return keep->const_data_ptr<T>();
}

// A [rows, n] operand with unit column stride (copied once if it has another).
Tensor matrix_of(const Tensor& t, int64_t rows, const Tensor& first, at::ScalarType type,
                 const char* name) {
  check_on(t, first, type, name);
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows, name, " must be 2-D with ", rows, " rows");
  return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous();
}

struct CacheArgs {
  int64_t pages, heads, page_size, dim, batch, max_pages;
  int dtype;
  Tensor table;
};

CacheArgs check_cache(const Tensor& k_cache, const Tensor& v_cache, const Tensor& table,
                      const Tensor& first) {
  TORCH_CHECK(k_cache.is_cuda(), "k_cache must be a CUDA tensor");
  TORCH_CHECK(k_cache.device() == first.device(), "k_cache must be on ", first.device());
  TORCH_CHECK(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes(),
              "k_cache, v_cache must be [pages, kv_heads, page_size, hs] of equal shape");
  check_on(v_cache, k_cache, k_cache.scalar_type(), "v_cache");
  check_on(table, k_cache, at::kInt, "block_table");
  TORCH_CHECK(table.dim() == 2, "block_table must be [batch, max_pages]");
  TORCH_CHECK(k_cache.stride(3) == 1 && v_cache.stride(3) == 1,
              "k_cache, v_cache must have unit stride along hs");
  CacheArgs a;
  a.pages = k_cache.size(0);
  a.heads = k_cache.size(1);
  a.page_size = k_cache.size(2);
  a.dim = k_cache.size(3);
  a.batch = table.size(0);
  a.max_pages = table.size(1);
  a.dtype = dtype_code(k_cache, "k_cache");
  a.table = table.stride(1) == 1 || a.max_pages <= 1 ? table : table.contiguous();
  return a;
}

void strides3(const Tensor& t, int64_t out[3]) {
  for (int i = 0; i < 3; ++i) out[i] = t.stride(i);
}

Tensor unit_last(const Tensor& t) { return t.stride(2) == 1 ? t : t.contiguous(); }

// One new token's keys and values (and queries) into / beside the cache.
std::tuple<Tensor, Tensor> kv_append_(Tensor k_cache, Tensor v_cache, Tensor k0, Tensor v0,
                                      Tensor table0, Tensor positions,
                                      std::optional<Tensor> seq_ids0, std::optional<Tensor> q0,
                                      std::optional<Tensor> cos0, std::optional<Tensor> sin0,
                                      bool interleaved, bool want_k,
                                      std::optional<Tensor> rotary_positions0) {
  const CacheArgs c = check_cache(k_cache, v_cache, table0, k0);
  const int act = dtype_code(k0, "k");
  check_on(v0, k0, k0.scalar_type(), "v");
  TORCH_CHECK(act == c.dtype || act == CT_DTYPE_F32, "k, v must be float32 or of the cache's type");
  TORCH_CHECK(k0.dim() == 3 && v0.sizes() == k0.sizes() && k0.size(1) == c.heads &&
                  k0.size(2) == c.dim,
              "k, v must be [tokens, kv_heads, hs]");
  c10::cuda::CUDAGuard guard(k0.device());
  const int64_t tokens = k0.size(0);
  const Tensor k = unit_last(k0), v = unit_last(v0);
  Tensor keep_pos, keep_seq, keep_rotary, q, cos, sin;
  const int32_t* pos = vector_of<int32_t>(positions, tokens, k, at::kInt, "positions", &keep_pos);
  const int32_t* seq = vector_of<int32_t>(seq_ids0, tokens, k, at::kInt, "seq_ids", &keep_seq);
  const int32_t* rotary = vector_of<int32_t>(rotary_positions0, tokens, k, at::kInt,
                                             "rotary_positions", &keep_rotary);
  int64_t q_heads = 0, rot = 0, max_positions = 0;
  int64_t qs[3] = {0, 0, 1}, ks[3], vs[3], kcs[4], vcs[4];
  if (q0.has_value()) {
    check_on(*q0, k, k.scalar_type(), "q");
    TORCH_CHECK(q0->dim() == 3 && q0->size(0) == tokens && q0->size(2) == c.dim,
                "q must be [tokens, nh, hs]");
    q = unit_last(*q0);
    q_heads = q.size(1);
    strides3(q, qs);
  }
  Tensor q_out = q0.has_value() ? empty_like_of({tokens, q_heads, c.dim}, k.scalar_type(), k)
                                : empty_like_of({0}, k.scalar_type(), k);
  Tensor k_out = want_k ? empty_like_of({tokens, c.heads, c.dim}, k.scalar_type(), k)
                        : empty_like_of({0}, k.scalar_type(), k);
  TORCH_CHECK(cos0.has_value() == sin0.has_value(), "cos and sin go together");
  if (cos0.has_value()) {
    check_on(*cos0, k, at::kFloat, "cos");
    check_on(*sin0, k, at::kFloat, "sin");
    TORCH_CHECK(cos0->dim() == 2 && sin0->sizes() == cos0->sizes() && 2 * cos0->size(1) <= c.dim,
                "cos, sin must be [positions, rot/2] of equal shape, rot <= hs");
    cos = cos0->contiguous();
    sin = sin0->contiguous();
    rot = 2 * cos.size(1);
    max_positions = cos.size(0);
  }
  strides3(k, ks);
  strides3(v, vs);
  strides4(k_cache, kcs);
  strides4(v_cache, vcs);
  check_rc(ct_kv_append_ex(q_heads ? q.const_data_ptr() : nullptr, qs, k.const_data_ptr(), ks,
                        v.const_data_ptr(), vs, q_heads ? q_out.data_ptr() : nullptr,
                        want_k ? k_out.data_ptr() : nullptr,
                        rot ? cos.const_data_ptr<float>() : nullptr,
                        rot ? sin.const_data_ptr<float>() : nullptr, k_cache.data_ptr(), kcs,
                        v_cache.data_ptr(), vcs, c.table.const_data_ptr<int32_t>(),
                        c.table.stride(0), seq, pos, rotary, tokens, q_heads, c.heads, c.dim, rot,
                        interleaved ? 1 : 0, max_positions, c.batch, c.pages, c.page_size,
                        c.max_pages, act, c.dtype, cur_stream()),
           "kv_append_");
  return {q_out, k_out};
}

int64_t paged_attention_workspace_size(int64_t nh, int64_t kv_heads, int64_t hs) {
  return (int64_t)ct_paged_attention_workspace_size(nh, kv_heads, hs);
}

std::tuple<Tensor, Tensor> paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor table,
                                           Tensor seq_lens, double scale,
                                           std::optional<Tensor> workspace) {
  const CacheArgs c = check_cache(k_cache, v_cache, table, q);
  const int act = dtype_code(q, "q");
  TORCH_CHECK(act == c.dtype || act == CT_DTYPE_F32, "q must be float32 or of the cache's type");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == c.dim, "q must be [batch, nh, hs]");
  TORCH_CHECK(q.size(0) == c.batch, "block_table must have a row for each row of q");
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t batch = q.size(0), heads = q.size(1);
  Tensor keep_lens;
  const int32_t* lens = vector_of<int32_t>(seq_lens, batch, q, at::kInt, "seq_lens", &keep_lens);
  const int64_t need = paged_attention_workspace_size(heads, c.heads, c.dim);
  Tensor ws;
  if (workspace.has_value()) {
    ws = *workspace;
    check_on(ws, q, at::kByte, "workspace");
    TORCH_CHECK(ws.is_contiguous() && ws.numel() >= need, "workspace must be dense, of ", need,
                " bytes or more");
  } else {
    // only the counters at its start have to be clear
    ws = empty_like_of({need}, at::kByte, q);
    ws.narrow(0, 0, CT_PAGED_ATTENTION_COUNTER_BYTES).zero_();
  }
  Tensor out = empty_like_of({batch, heads, c.dim}, q.scalar_type(), q);
  Tensor lse = empty_like_of({batch, heads}, at::kFloat, q);
  int64_t qs[3], kcs[4], vcs[4];
  strides3(q, qs);
  strides4(k_cache, kcs);
  strides4(v_cache, vcs);
  check_rc(ct_paged_attention(q.const_data_ptr(), qs, k_cache.const_data_ptr(), kcs,
                              v_cache.const_data_ptr(), vcs, c.table.const_data_ptr<int32_t>(),
                              c.table.stride(0), lens, out.data_ptr(), lse.data_ptr<float>(),
                              batch, heads, c.heads, c.dim, c.pages, c.page_size, c.max_pages,
                              (float)scale, act, c.dtype, ws.data_ptr(), (size_t)ws.numel(),
                              cur_stream()),
           "paged_attention");
  return {out, lse};
}

Tensor logits_process(Tensor logits0, std::optional<Tensor> tokens0, std::optional<Tensor> lens0,
                      std::optional<Tensor> prompt_lens0, std::optional<Tensor> repetition0,
                      std::optional<Tensor> frequency0, std::optional<Tensor> presence0,
                      std::optional<Tensor> bias_ids0, std::optional<Tensor> bias_values0,
                      std::optional<Tensor> mask0) {
  TORCH_CHECK(logits0.is_cuda(), "logits must be a CUDA tensor");
  TORCH_CHECK(logits0.dim() == 2, "logits must be (rows, vocab)");
  const int dtype = dtype_code(logits0, "logits");
  c10::cuda::CUDAGuard guard(logits0.device());
  const int64_t rows = logits0.size(0), vocab = logits0.size(1);
  Tensor logits = matrix_of(logits0, rows, logits0, logits0.scalar_type(), "logits");
  if (rows > 1 && logits.stride(0) < vocab) logits = logits.contiguous();  // a broadcast row
  Tensor keep[5], tokens, ids, values, mask;
  if (tokens0.has_value()) tokens = matrix_of(*tokens0, rows, logits, at::kLong, "tokens");
  const int32_t* lens = vector_of<int32_t>(lens0, rows, logits, at::kInt, "lens", &keep[0]);
  const int32_t* plens =
      vector_of<int32_t>(prompt_lens0, rows, logits, at::kInt, "prompt_lens", &keep[1]);
  const float* rep =
      vector_of<float>(repetition0, rows, logits, at::kFloat, "repetition", &keep[2]);
  const float* freq = vector_of<float>(frequency0, rows, logits, at::kFloat, "frequency", &keep[3]);
  const float* pres = vector_of<float>(presence0, rows, logits, at::kFloat, "presence", &keep[4]);
  TORCH_CHECK(bias_ids0.has_value() == bias_values0.has_value(),
              "bias_ids and bias_values go together");
  int64_t bias_n = 0;
  if (bias_ids0.has_value()) {
    ids = matrix_of(*bias_ids0, rows, logits, at::kLong, "bias_ids");
    values = matrix_of(*bias_values0, rows, logits, at::kFloat, "bias_values");
    bias_n = ids.size(1);
    TORCH_CHECK(values.size(1) == bias_n, "bias_values must have bias_ids' shape");
  }
  if (mask0.has_value()) {
    mask = matrix_of(*mask0, rows, logits, at::kInt, "mask");
    TORCH_CHECK(mask.size(1) >= (vocab + 31) / 32, "mask must have ceil(vocab / 32) words a row");
  }
  Tensor out = empty_like_of({rows, vocab}, at::kFloat, logits);
  check_rc(ct_logits_process(logits.const_data_ptr(), rows > 1 ? logits.stride(0) : vocab, dtype,
                             out.data_ptr<float>(), vocab, rows, vocab,
                             tokens.defined() ? tokens.const_data_ptr<int64_t>() : nullptr,
                             tokens.defined() ? tokens.stride(0) : 0,
                             tokens.defined() ? tokens.size(1) : 0, lens, plens, rep, freq, pres,
                             bias_n ? ids.const_data_ptr<int64_t>() : nullptr,
                             bias_n ? ids.stride(0) : 0,
                             bias_n ? values.const_data_ptr<float>() : nullptr,
                             bias_n ? values.stride(0) : 0, bias_n,
                             mask.defined() ? mask.const_data_ptr<int32_t>() : nullptr,
                             mask.defined() ? mask.stride(0) : 0, cur_stream()),
           "logits_process");
  return out;
}

// ------------------------------------------------------ speculative decoding
std::tuple<Tensor, Tensor> tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor table,
                                          Tensor context_lens0, std::optional<Tensor> draft_lens0,
                                          std::optional<Tensor> mask0, double scale) {
  const CacheArgs c = check_cache(k_cache, v_cache, table, q);
  const int act = dtype_code(q, "q");
  TORCH_CHECK(act == c.dtype || act == CT_DTYPE_F32, "q must be float32 or of the cache's type");
  TORCH_CHECK(q.dim() == 4 && q.size(3) == c.dim, "q must be [batch, drafts, nh, hs]");
  TORCH_CHECK(q.size(0) == c.batch, "block_table must have a row for each sequence of q");
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t batch = q.size(0), drafts = q.size(1), heads = q.size(2);
  Tensor keep_context, keep_drafts, mask;
  const int32_t* context =
      vector_of<int32_t>(context_lens0, batch, q, at::kInt, "context_lens", &keep_context);
  const int32_t* lens =
      vector_of<int32_t>(draft_lens0, batch, q, at::kInt, "draft_lens", &keep_drafts);
  int64_t ms[2] = {0, 0};
  if (mask0.has_value()) {
    mask = *mask0;
    check_on(mask, q, at::kInt, "mask");
    TORCH_CHECK(mask.dim() == 3 && mask.size(0) == batch && mask.size(1) == drafts &&
                    mask.size(2) >= (drafts + 31) / 32,
                "mask must be [batch, drafts, ceil(drafts / 32)]");
    if (mask.stride(2) != 1 && mask.size(2) > 1) mask = mask.contiguous();
    ms[0] = mask.stride(0);
    ms[1] = mask.stride(1);
  }
  const int64_t need = ct_tree_attention_workspace_size(drafts, heads, c.heads, c.dim);
  // (no counters in it: nothing to clear, and a captured call has its own)
  Tensor ws = empty_like_of({need}, at::kByte, q);
  Tensor out = empty_like_of({batch, drafts, heads, c.dim}, q.scalar_type(), q);
  Tensor lse = empty_like_of({batch, drafts, heads}, at::kFloat, q);
  int64_t qs[4], kcs[4], vcs[4];
  strides4(q, qs);
  strides4(k_cache, kcs);
  strides4(v_cache, vcs);
  check_rc(ct_tree_attention(q.const_data_ptr(), qs, k_cache.const_data_ptr(), kcs,
                             v_cache.const_data_ptr(), vcs, c.table.const_data_ptr<int32_t>(),
                             c.table.stride(0), context, lens,
                             mask.defined() ? mask.const_data_ptr<int32_t>() : nullptr, ms,
                             out.data_ptr(), lse.data_ptr<float>(), batch, drafts, heads, c.heads,
                             c.dim, c.pages, c.page_size, c.max_pages, (float)scale, act, c.dtype,
                             ws.data_ptr(), (size_t)need, cur_stream()),
           "tree_attention");
  return {out, lse};
}

// [batch, nodes, vocab] with unit stride along the last (copied once otherwise).
Tensor node_rows(const Tensor& t, const Tensor& first, at::ScalarType type, const char* name) {
  check_on(t, first, type, name);
  TORCH_CHECK(t.dim() == 3 && t.sizes() == first.sizes(), name,
              " must be [batch, drafts, vocab], as target");
  return t.stride(2) == 1 || t.size(2) <= 1 ? t : t.contiguous();
}

std::tuple<Tensor, Tensor, Tensor> verify_drafts(Tensor target0, Tensor tokens0,
                                                 std::optional<Tensor> parents0,
                                                 std::optional<Tensor> draft_lens0,
                                                 std::optional<Tensor> draft_probs0,
                                                 std::optional<Tensor> uniform0) {
  TORCH_CHECK(target0.is_cuda(), "target must be a CUDA tensor");
  const int dtype = dtype_code(target0, "target");
  const Tensor target = node_rows(target0, target0, target0.scalar_type(), "target");
  c10::cuda::CUDAGuard guard(target.device());
  const int64_t batch = target.size(0), drafts = target.size(1), vocab = target.size(2);
  TORCH_CHECK(!draft_probs0.has_value() || uniform0.has_value(), "draft_probs needs uniform");
  auto of_nodes = [&](const Tensor& t, at::ScalarType type, const char* name) {
    Tensor m = matrix_of(t, batch, target, type, name);
    TORCH_CHECK(m.size(1) == drafts, name, " must be [batch, drafts]");
    return m;
  };
  const Tensor tokens = of_nodes(tokens0, at::kLong, "tokens");
  Tensor parents, uniform, draft_probs, keep_lens;
  if (parents0.has_value()) parents = of_nodes(*parents0, at::kInt, "parents");
  if (uniform0.has_value()) uniform = of_nodes(*uniform0, at::kFloat, "uniform");
  if (draft_probs0.has_value())
    draft_probs = node_rows(*draft_probs0, target, target.scalar_type(), "draft_probs");
  const int32_t* lens =
      vector_of<int32_t>(draft_lens0, batch, target, at::kInt, "draft_lens", &keep_lens);
  Tensor new_tokens = empty_like_of({batch, drafts}, at::kLong, target);
  Tensor path = empty_like_of({batch, drafts}, at::kInt, target);
  Tensor counts = empty_like_of({batch}, at::kInt, target);
  const int64_t ts[2] = {target.stride(0), target.stride(1)};
  int64_t ds[2] = {0, 0};
  if (draft_probs.defined()) {
    ds[0] = draft_probs.stride(0);
    ds[1] = draft_probs.stride(1);
  }
  check_rc(ct_verify_drafts(target.const_data_ptr(), ts,
                            draft_probs.defined() ? draft_probs.const_data_ptr() : nullptr, ds,
                            dtype, tokens.const_data_ptr<int64_t>(), tokens.stride(0),
                            parents.defined() ? parents.const_data_ptr<int32_t>() : nullptr,
                            parents.defined() ? parents.stride(0) : 0, lens,
                            uniform.defined() ? uniform.const_data_ptr<float>() : nullptr,
                            uniform.defined() ? uniform.stride(0) : 0,
                            new_tokens.data_ptr<int64_t>(), path.data_ptr<int32_t>(),
                            counts.data_ptr<int32_t>(), batch, drafts, vocab, cur_stream()),
           "verify_drafts");
  return {new_tokens, path, counts};
}

// A list of caches of one shape and type, as the C ABI takes it.
struct CacheTensors {
  std::vector<void*> base;
  std::vector<int64_t> strides;
  int64_t pages = 0, heads = 1, page_size = 1, dim = 1;
  int dtype = CT_DTYPE_F32;
};

CacheTensors cache_tensors(at::TensorList caches) {
  CacheTensors c;
  for (const Tensor& t : caches) {
    TORCH_CHECK(t.is_cuda(), "caches must be CUDA tensors");
    check_on(t, caches[0], caches[0].scalar_type(), "caches");
    TORCH_CHECK(t.dim() == 4 && t.sizes() == caches[0].sizes(),
                "caches must be [pages, kv_heads, page_size, hs] of equal shape");
    TORCH_CHECK(t.stride(3) == 1 || t.size(3) <= 1, "caches must have unit stride along hs");
    c.base.push_back(t.data_ptr());
    for (int i = 0; i < 4; ++i) c.strides.push_back(t.stride(i));
  }
  if (!caches.empty()) {
    c.pages = caches[0].size(0);
    c.heads = caches[0].size(1);
    c.page_size = caches[0].size(2);
    c.dim = caches[0].size(3);
    c.dtype = dtype_code(caches[0], "caches");
  }
  return c;
}

void kv_compact_(at::TensorList caches, Tensor table0, Tensor context_lens0, Tensor keep0,
                 Tensor counts0) {
  TORCH_CHECK(!caches.empty(), "caches must not be an empty list");
  const CacheTensors c = cache_tensors(caches);
  c10::cuda::CUDAGuard guard(caches[0].device());
  const int64_t batch = table0.size(0);
  const Tensor table = matrix_of(table0, batch, caches[0], at::kInt, "block_table");
  const Tensor keep = matrix_of(keep0, batch, caches[0], at::kInt, "keep");
  Tensor keep_context, keep_counts;
  const int32_t* context = vector_of<int32_t>(context_lens0, batch, caches[0], at::kInt,
                                              "context_lens", &keep_context);
  const int32_t* counts =
      vector_of<int32_t>(counts0, batch, caches[0], at::kInt, "counts", &keep_counts);
  check_rc(ct_kv_compact(c.base.data(), c.strides.data(), (int64_t)c.base.size(),
                         table.const_data_ptr<int32_t>(), table.stride(0), context,
                         keep.const_data_ptr<int32_t>(), keep.stride(0), counts, batch,
                         keep.size(1), c.heads, c.dim, c.pages, c.page_size, table.size(1),
                         c.dtype, cur_stream()),
           "kv_compact_");
}

void kv_copy_pages_(at::TensorList caches, Tensor src0, Tensor dst0) {
  TORCH_CHECK(!caches.empty(), "caches must not be an empty list");
  const CacheTensors c = cache_tensors(caches);
  c10::cuda::CUDAGuard guard(caches[0].device());
  const int64_t n = src0.numel();
  Tensor keep_src, keep_dst;
  const int32_t* src = vector_of<int32_t>(src0, n, caches[0], at::kInt, "src", &keep_src);
  const int32_t* dst = vector_of<int32_t>(dst0, n, caches[0], at::kInt, "dst", &keep_dst);
  check_rc(ct_kv_copy_pages(c.base.data(), c.strides.data(), (int64_t)c.base.size(), src, dst, n,
                            c.heads, c.dim, c.pages, c.page_size, c.dtype, cur_stream()),
           "kv_copy_pages_");
}

// ------------------------------------------- materialised (naive) attention
// Kept registered so cuda_autograd_fns imports; composed from this library's
// own GEMM and softmax kernels.  qkv: (B, T, 3C) contiguous.
std::tuple<Tensor, Tensor> causal_self_attention_fwd(Tensor qkv, int64_t nh, bool causal) {
  check_cuda_f32(qkv, "qkv");
  TORCH_CHECK(qkv.is_contiguous(), "qkv must be contiguous");
  TORCH_CHECK(qkv.dim() == 3 && qkv.size(2) % (3 * nh) == 0, "qkv must be (B, T, 3*nh*hs)");
  c10::cuda::CUDAGuard guard(qkv.device());
  const int64_t B = qkv.size(0), T = qkv.size(1), C = qkv.size(2) / 3, hs = C / nh;
  const int prec = default_precision();
  auto heads = [&](int64_t part) {  // (B*nh, T, hs) view of one third of qkv
    return qkv.narrow(2, part * C, C).reshape({B, T, nh, hs}).transpose(1, 2).reshape({B * nh, T, hs});
  };
  Tensor q = heads(0), k = heads(1), v = heads(2);
  Tensor zero_t = at::zeros({T}, qkv.options());
  // S = q k^T / sqrt(hs): weights = k^T viewed (B*nh, hs, T)
  Tensor s = fma_impl(q, k.transpose(1, 2), zero_t, prec).mul_(1.0 / std::sqrt((double)hs));
  if (causal) s.masked_fill_(at::ones({T, T}, qkv.options().dtype(at::kBool)).triu(1), -INFINITY);
  Tensor probs = at::empty_like(s);
  check_rc(ct_softmax_fwd(s.data_ptr<float>(), probs.data_ptr<float>(), B * nh * T, T, cur_stream()),
           "causal_self_attention_fwd");
  Tensor zero_h = at::zeros({hs}, qkv.options());
  Tensor o = fma_impl(probs, v, zero_h, prec);  // (B*nh, T, hs)
  Tensor out = o.reshape({B, nh, T, hs}).transpose(1, 2).reshape({B, T, C}).contiguous();
  return {out, probs.reshape({B, nh, T, T})};
}

// Gradients with the test's convention (test/test_causal_self_attn.py:60-67):
// returns dq and dk multiplied by sqrt(hs) and dv unscaled.
std::tuple<Tensor, Tensor, Tensor> causal_self_attention_bwd(Tensor Q, Tensor K, Tensor V,
                                                             Tensor probs, Tensor dO) {
  check_cuda_f32(Q, "Q");
  check_cuda_f32(K, "K");
  check_cuda_f32(V, "V");
  check_cuda_f32(probs, "probs");
  check_cuda_f32(dO, "dO");
  c10::cuda::CUDAGuard guard(Q.device());
  const int64_t BH = Q.size(0), T = Q.size(1), hs = Q.size(2);
  const int prec = default_precision();
  Tensor P = probs.reshape({BH, T, T}).contiguous();
  Tensor zT = at::zeros({T}, Q.options()), zH = at::zeros({hs}, Q.options());
  Tensor dV = fma_impl(P.transpose(1, 2), dO, zH, prec);         // P^T dO
  Tensor dP = fma_impl(dO, V.transpose(1, 2), zT, prec);         // dO V^T
  Tensor dS = at::empty_like(P);
  check_rc(ct_softmax_bwd(P.data_ptr<float>(), dP.contiguous().data_ptr<float>(),
                          dS.data_ptr<float>(), BH * T, T, cur_stream()),
           "causal_self_attention_bwd");
  Tensor dQ = fma_impl(dS, K, zH, prec);                          // dS K
  Tensor dK = fma_impl(dS.transpose(1, 2), Q, zH, prec);          // dS^T Q
  return {dQ, dK, dV};
}

}  // namespace

TORCH_LIBRARY(cuda_transformer, m) {
  m.def("cuda_fma(Tensor x, Tensor weights, Tensor bias) -> Tensor");
  m.def("db_calculation(Tensor dy) -> Tensor");
  m.def("cuda_softmax(Tensor x) -> Tensor");
  m.def("cuda_softmax_bwd(Tensor probs, Tensor dp) -> Tensor");
  m.def("gelu_activation(Tensor x) -> Tensor");
  m.def("gelu_activation_bwd(Tensor x, Tensor dy) -> Tensor");
  m.def("flash_attention_fwd(Tensor Q, Tensor K, Tensor V, bool causal) -> (Tensor, Tensor)");
  m.def("flash_attention_bwd(Tensor Q, Tensor K, Tensor V, Tensor O, Tensor dO, Tensor L, bool causal) -> (Tensor, Tensor, Tensor)");
  m.def("causal_self_attention_fwd(Tensor qkv, int nh, bool causal) -> (Tensor, Tensor)");
  m.def("causal_self_attention_bwd(Tensor Q, Tensor K, Tensor V, Tensor probs, Tensor dO) -> (Tensor, Tensor, Tensor)");
  // additions of this implementation
  m.def("flash_attention_fwd_ex(Tensor Q, Tensor K, Tensor V, bool causal, int precision) -> (Tensor, Tensor)");
  m.def("flash_attention_bwd_ex(Tensor Q, Tensor K, Tensor V, Tensor O, Tensor dO, Tensor L, bool causal, int precision) -> (Tensor, Tensor, Tensor)");
  m.def("cuda_fma_ex(Tensor x, Tensor weights, Tensor bias, int precision) -> Tensor");
  m.def("layernorm_fwd(Tensor x, Tensor gamma, Tensor beta, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("layernorm_bwd(Tensor x, Tensor gamma, Tensor mean, Tensor rstd, Tensor dy) -> (Tensor, Tensor, Tensor)");
  m.def("linear_fused(Tensor x, Tensor weights, Tensor bias, int precision, int epilogue, Tensor? act_in, bool want_colsum) -> (Tensor, Tensor, Tensor)");
  m.def("linear_accumulate_(Tensor(a!) out, Tensor(b!)? colsum, Tensor x, Tensor weights, Tensor bias, int precision) -> ()");
  m.def("cross_entropy_fwd_bwd_(Tensor(a!) logits, Tensor targets, int ignore_index) -> Tensor");
  m.def("kv_append_(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor k, Tensor v, Tensor block_table, Tensor positions, Tensor? seq_ids, Tensor? q, Tensor? cos, Tensor? sin, bool interleaved, bool want_k, Tensor? rotary_positions=None) -> (Tensor, Tensor)");
  m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens, float scale, Tensor(a!)? workspace) -> (Tensor, Tensor)");
  m.def("paged_attention_workspace_size(int nh, int kv_heads, int hs) -> int", &paged_attention_workspace_size);
  m.def("logits_process(Tensor logits, Tensor? tokens, Tensor? lens, Tensor? prompt_lens, Tensor? repetition, Tensor? frequency, Tensor? presence, Tensor? bias_ids, Tensor? bias_values, Tensor? mask) -> Tensor");
  m.def("tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor context_lens, Tensor? draft_lens, Tensor? mask, float scale) -> (Tensor, Tensor)");
  m.def("verify_drafts(Tensor target, Tensor tokens, Tensor? parents, Tensor? draft_lens, Tensor? draft_probs, Tensor? uniform) -> (Tensor, Tensor, Tensor)");
  m.def("kv_compact_(Tensor(a!)[] caches, Tensor block_table, Tensor context_lens, Tensor keep, Tensor counts) -> ()");
  m.def("kv_copy_pages_(Tensor(a!)[] caches, Tensor src, Tensor dst) -> ()");
}

TORCH_LIBRARY_IMPL(cuda_transformer, CUDA, m) {
  m.impl("cuda_fma", &cuda_fma);
  m.impl("db_calculation", &db_calculation);
  m.impl("cuda_softmax", &cuda_softmax);
  m.impl("cuda_softmax_bwd", &cuda_softmax_bwd);
  m.impl("gelu_activation", &gelu_activation);
  m.impl("gelu_activation_bwd", &gelu_activation_bwd);
  m.impl("flash_attention_fwd", &flash_attention_fwd);
  m.impl("flash_attention_bwd", &flash_attention_bwd);
  m.impl("causal_self_attention_fwd", &causal_self_attention_fwd);
  m.impl("causal_self_attention_bwd", &causal_self_attention_bwd);
  m.impl("flash_attention_fwd_ex", &flash_attention_fwd_ex);
  m.impl("flash_attention_bwd_ex", &flash_attention_bwd_ex);
  m.impl("cuda_fma_ex", &cuda_fma_ex);
  m.impl("layernorm_fwd", &layernorm_fwd);
  m.impl("layernorm_bwd", &layernorm_bwd);
  m.impl("linear_fused", &linear_fused);
  m.impl("linear_accumulate_", &linear_accumulate_);
  m.impl("cross_entropy_fwd_bwd_", &cross_entropy_fwd_bwd_);
  m.impl("kv_append_", &kv_append_);
  m.impl("paged_attention", &paged_attention);
  m.impl("logits_process", &logits_process);
  m.impl("tree_attention", &tree_attention);
  m.impl("verify_drafts", &verify_drafts);
  m.impl("kv_compact_", &kv_compact_);
  m.impl("kv_copy_pages_", &kv_copy_pages_);
}

}  // namespace cuda_transformer

// Python module object for `import cuda_transformer._C`; loading the shared
// object runs the static operator registrations above.
static PyModuleDef ct_module = {PyModuleDef_HEAD_INIT, "_C",
                                "custom cuda kernels for transformer architecture (sm_100a)", -1,
                                nullptr};
PyMODINIT_FUNC PyInit__C(void) { return PyModule_Create(&ct_module); }
