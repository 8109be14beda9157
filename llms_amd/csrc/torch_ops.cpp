// torch_ops.cpp — the thin PyTorch-ROCm custom ops over the C ABI of
// include/llms_amd_fp.h. Each op allocates its output (and, for the bf16
// calls that split k across workgroups, the workspace) with torch on the
// tensor's device, takes torch's current HIP stream, and hands plain pointers,
// row strides and sizes to the C ABI; a nonzero fp_status becomes a
// c10::Error (RuntimeError in Python). No computation happens here.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include "llms_amd_fp.h"

namespace {

void check_status(int st, const char* fn) {
  TORCH_CHECK(st == FP_OK, fn, " failed: ", fp_status_string(st), " (fp_status ", st, ")");
}

void check_2d(const at::Tensor& t, const char* name, at::ScalarType dt) {
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D, got ", t.dim(), "-D");
  TORCH_CHECK(t.scalar_type() == dt, name, " must be ", c10::toString(dt), ", got ",
              c10::toString(t.scalar_type()));
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have unit inner stride");
  TORCH_CHECK(t.is_cuda(), name, " must be a HIP device tensor");
}

// Every tensor of a call lives on x's device (the kernels dereference all of
// them there; a host pointer would fault the GPU).
void check_same_device(const at::Tensor& x, const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), name, " must be on ", x.device(),
              ", got ", t.device());
}

// A weight [N, K] of the call: K columns (the x row length), on x's device.
void check_weight(const at::Tensor& x, const at::Tensor& w, const char* name) {
  TORCH_CHECK(w.size(1) == x.size(1), name, " has ", w.size(1), " columns, x has K = ",
              x.size(1));
  check_same_device(x, w, name);
}

// Per-row int8 scales of weight q: contiguous 1-D fp32, one per row, on x's
// device.
void check_scale(const at::Tensor& x, const at::Tensor& s, const at::Tensor& q, const char* name) {
  TORCH_CHECK(s.dim() == 1 && s.scalar_type() == at::kFloat && s.is_contiguous(), name,
              " must be a contiguous 1-D float32 tensor");
  TORCH_CHECK(s.size(0) == q.size(0), name, " has ", s.size(0), " rows, q has ", q.size(0));
  check_same_device(x, s, name);
}

// Gate and up weights of one call have the same shape.
void check_pair(const at::Tensor& g, const at::Tensor& u, const char* gn, const char* un) {
  TORCH_CHECK(g.sizes() == u.sizes(), gn, " ", g.sizes(), " and ", un, " ", u.sizes(),
              " must have the same shape");
}

void* cur_stream(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// Split-k workspace for a bf16 call, from torch's caching allocator on the
// current stream (empty when the call does not split).
at::Tensor workspace(const at::Tensor& x, int64_t M, int64_t N, int64_t K, bool gate_up) {
  const int64_t bytes = fp_workspace_bytes(M, N, K, gate_up ? 1 : 0);
  return at::empty({bytes}, x.options().dtype(at::kByte));
}

// Workspace for an int8 call: the fp32 partials where k is split across
// workgroups, empty otherwise (int8 weights are never expanded to bf16).
at::Tensor workspace_w8(const at::Tensor& x, int64_t M, int64_t N, int64_t K, bool gate_up) {
  const int64_t bytes = fp_workspace_bytes_w8(M, N, K, gate_up ? 1 : 0);
  return at::empty({bytes}, x.options().dtype(at::kByte));
}

at::Tensor qkv(const at::Tensor& x, const at::Tensor& w, int64_t n_q, int64_t n_k) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(w, "W_qkv", at::kBFloat16);
  check_weight(x, w, "W_qkv");
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = workspace(x, M, N, K, false);
  check_status(fp_qkv_bf16_ws(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), y.data_ptr(),
                              y.stride(0), M, n_q, n_k, K, ws.numel() ? ws.data_ptr() : nullptr,
                              ws.numel(), cur_stream(x)),
               "fp_qkv_bf16_ws");
  return y;
}

at::Tensor gate_up_silu(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(wg, "Wg", at::kBFloat16);
  check_2d(wu, "Wu", at::kBFloat16);
  check_weight(x, wg, "Wg");
  check_weight(x, wu, "Wu");
  check_pair(wg, wu, "Wg", "Wu");
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = wg.size(0);
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = workspace(x, M, N, K, true);
  check_status(fp_gate_up_silu_bf16_ws(x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0),
                                       wu.data_ptr(), wu.stride(0), y.data_ptr(), y.stride(0), M,
                                       N, K, ws.numel() ? ws.data_ptr() : nullptr, ws.numel(),
                                       cur_stream(x)),
               "fp_gate_up_silu_bf16_ws");
  return y;
}

at::Tensor qkv_w8(const at::Tensor& x, const at::Tensor& q, const at::Tensor& s, int64_t n_q,
                  int64_t n_k) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(q, "q", at::kChar);
  check_weight(x, q, "q");
  check_scale(x, s, q, "scale");
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = q.size(0);
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = workspace_w8(x, M, N, K, false);
  check_status(fp_qkv_w8_ws(x.data_ptr(), x.stride(0), (const int8_t*)q.data_ptr(), q.stride(0),
                            s.data_ptr<float>(), y.data_ptr(), y.stride(0), M, n_q, n_k, K,
                            ws.numel() ? ws.data_ptr() : nullptr, ws.numel(), cur_stream(x)),
               "fp_qkv_w8_ws");
  return y;
}

at::Tensor gate_up_silu_w8(const at::Tensor& x, const at::Tensor& qg, const at::Tensor& sg,
                           const at::Tensor& qu, const at::Tensor& su) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(qg, "qg", at::kChar);
  check_2d(qu, "qu", at::kChar);
  check_weight(x, qg, "qg");
  check_weight(x, qu, "qu");
  check_pair(qg, qu, "qg", "qu");
  check_scale(x, sg, qg, "sg");
  check_scale(x, su, qu, "su");
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = qg.size(0);
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = workspace_w8(x, M, N, K, true);
  check_status(fp_gate_up_silu_w8_ws(x.data_ptr(), x.stride(0), (const int8_t*)qg.data_ptr(),
                                     qg.stride(0), sg.data_ptr<float>(),
                                     (const int8_t*)qu.data_ptr(), qu.stride(0),
                                     su.data_ptr<float>(), y.data_ptr(), y.stride(0), M, N, K,
                                     ws.numel() ? ws.data_ptr() : nullptr, ws.numel(),
                                     cur_stream(x)),
               "fp_gate_up_silu_w8_ws");
  return y;
}

at::Tensor linear(const at::Tensor& x, const at::Tensor& w) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(w, "W", at::kBFloat16);
  check_weight(x, w, "W");
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = workspace(x, M, N, K, false);
  check_status(fp_linear_bf16_ws(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0),
                                 y.data_ptr(), y.stride(0), M, N, K,
                                 ws.numel() ? ws.data_ptr() : nullptr, ws.numel(), cur_stream(x)),
               "fp_linear_bf16_ws");
  return y;
}

at::Tensor linear_w8(const at::Tensor& x, const at::Tensor& q, const at::Tensor& s) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(q, "q", at::kChar);
  check_weight(x, q, "q");
  check_scale(x, s, q, "scale");
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = q.size(0);
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = workspace_w8(x, M, N, K, false);
  check_status(fp_linear_w8_ws(x.data_ptr(), x.stride(0), (const int8_t*)q.data_ptr(), q.stride(0),
                               s.data_ptr<float>(), y.data_ptr(), y.stride(0), M, N, K,
                               ws.numel() ? ws.data_ptr() : nullptr, ws.numel(), cur_stream(x)),
               "fp_linear_w8_ws");
  return y;
}

// ---- RMSNorm prologue fused with the projections ----

void check_gamma(const at::Tensor& x, const at::Tensor& gamma) {
  TORCH_CHECK(gamma.dim() == 1 && gamma.scalar_type() == at::kBFloat16 && gamma.is_contiguous(),
              "norm weight must be a contiguous 1-D bfloat16 tensor");
  TORCH_CHECK(gamma.size(0) == x.size(1), "norm weight has ", gamma.size(0),
              " elements, x has K = ", x.size(1));
  check_same_device(x, gamma, "norm weight");
}

// Workspace for a fused-norm call: what the library asks for (enough for any
// pointers and strides of the shape).
at::Tensor norm_workspace(const at::Tensor& x, int64_t M, int64_t N, int64_t K, bool gate_up,
                          bool int8) {
  const int64_t bytes = fp_rmsnorm_workspace_bytes(M, N, K, gate_up ? 1 : 0, int8 ? 1 : 0);
  return at::empty({bytes}, x.options().dtype(at::kByte));
}

at::Tensor rmsnorm_qkv(const at::Tensor& x, const at::Tensor& gamma, double eps,
                       const at::Tensor& w, int64_t n_q, int64_t n_k) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(w, "W_qkv", at::kBFloat16);
  check_weight(x, w, "W_qkv");
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  check_gamma(x, gamma);
  const c10::DeviceGuard guard(x.device());
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = norm_workspace(x, M, N, K, false, false);
  check_status(fp_rmsnorm_qkv_bf16(x.data_ptr(), x.stride(0), gamma.data_ptr(), (float)eps,
                                   w.data_ptr(), w.stride(0), y.data_ptr(), y.stride(0), M, n_q,
                                   n_k, K, ws.data_ptr(), ws.numel(), cur_stream(x)),
               "fp_rmsnorm_qkv_bf16");
  return y;
}

at::Tensor rmsnorm_gate_up_silu(const at::Tensor& x, const at::Tensor& gamma, double eps,
                                const at::Tensor& wg, const at::Tensor& wu) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(wg, "Wg", at::kBFloat16);
  check_2d(wu, "Wu", at::kBFloat16);
  check_weight(x, wg, "Wg");
  check_weight(x, wu, "Wu");
  check_pair(wg, wu, "Wg", "Wu");
  const int64_t M = x.size(0), K = x.size(1), N = wg.size(0);
  check_gamma(x, gamma);
  const c10::DeviceGuard guard(x.device());
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = norm_workspace(x, M, N, K, true, false);
  check_status(fp_rmsnorm_gate_up_silu_bf16(x.data_ptr(), x.stride(0), gamma.data_ptr(),
                                            (float)eps, wg.data_ptr(), wg.stride(0),
                                            wu.data_ptr(), wu.stride(0), y.data_ptr(),
                                            y.stride(0), M, N, K, ws.data_ptr(), ws.numel(),
                                            cur_stream(x)),
               "fp_rmsnorm_gate_up_silu_bf16");
  return y;
}

at::Tensor rmsnorm_qkv_w8(const at::Tensor& x, const at::Tensor& gamma, double eps,
                          const at::Tensor& q, const at::Tensor& s, int64_t n_q, int64_t n_k) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(q, "q", at::kChar);
  check_weight(x, q, "q");
  check_scale(x, s, q, "scale");
  const int64_t M = x.size(0), K = x.size(1), N = q.size(0);
  check_gamma(x, gamma);
  const c10::DeviceGuard guard(x.device());
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = norm_workspace(x, M, N, K, false, true);
  check_status(fp_rmsnorm_qkv_w8(x.data_ptr(), x.stride(0), gamma.data_ptr(), (float)eps,
                                 (const int8_t*)q.data_ptr(), q.stride(0), s.data_ptr<float>(),
                                 y.data_ptr(), y.stride(0), M, n_q, n_k, K, ws.data_ptr(),
                                 ws.numel(), cur_stream(x)),
               "fp_rmsnorm_qkv_w8");
  return y;
}

at::Tensor rmsnorm_gate_up_silu_w8(const at::Tensor& x, const at::Tensor& gamma, double eps,
                                   const at::Tensor& qg, const at::Tensor& sg,
                                   const at::Tensor& qu, const at::Tensor& su) {
  check_2d(x, "x", at::kBFloat16);
  check_2d(qg, "qg", at::kChar);
  check_2d(qu, "qu", at::kChar);
  check_weight(x, qg, "qg");
  check_weight(x, qu, "qu");
  check_pair(qg, qu, "qg", "qu");
  check_scale(x, sg, qg, "sg");
  check_scale(x, su, qu, "su");
  const int64_t M = x.size(0), K = x.size(1), N = qg.size(0);
  check_gamma(x, gamma);
  const c10::DeviceGuard guard(x.device());
  at::Tensor y = at::empty({M, N}, x.options());
  at::Tensor ws = norm_workspace(x, M, N, K, true, true);
  check_status(fp_rmsnorm_gate_up_silu_w8(x.data_ptr(), x.stride(0), gamma.data_ptr(),
                                          (float)eps, (const int8_t*)qg.data_ptr(), qg.stride(0),
                                          sg.data_ptr<float>(), (const int8_t*)qu.data_ptr(),
                                          qu.stride(0), su.data_ptr<float>(), y.data_ptr(),
                                          y.stride(0), M, N, K, ws.data_ptr(), ws.numel(),
                                          cur_stream(x)),
               "fp_rmsnorm_gate_up_silu_w8");
  return y;
}

// ---- the attention layer between its projections ----

// q [B, T, n] as rows b*T + t of a row stride the kernels take; -1 if not.
int64_t token_rows(const at::Tensor& t, int64_t B, int64_t T, int64_t n) {
  if (t.dim() != 3 || t.size(0) != B || t.size(1) != T || t.size(2) != n || t.stride(2) != 1)
    return -1;
  const int64_t ld = T > 1 ? t.stride(1) : B > 1 ? t.stride(0) : n;
  if (B > 1 && t.stride(0) != T * ld) return -1;
  return ld >= n && ld % 4 == 0 && (uintptr_t)t.data_ptr() % 8 == 0 ? ld : -1;
}

// q, k, v: the projection's flat outputs. q_gamma, k_gamma: the QK-norm
// weights, or absent where q and k are normalised already. Returns the
// attention output [B, T, n_heads * D], or an empty 1-D tensor, with nothing
// launched and nothing written, where the kernels do not take the call (types,
// devices, sizes, strides): the caller then runs the torch form, which also
// raises the errors of invalid calls.
at::Tensor attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                     const c10::optional<at::Tensor>& q_gamma,
                     const c10::optional<at::Tensor>& k_gamma, double q_eps, double k_eps,
                     const at::Tensor& cos, const at::Tensor& sin, at::Tensor cache_k,
                     at::Tensor cache_v, int64_t n_heads, int64_t start_pos,
                     const c10::optional<at::Tensor>& pos) {
  const auto none = [&] { return at::empty({0}, q.options()); };
  const auto bf16_here = [&](const at::Tensor& t) {
    return t.scalar_type() == at::kBFloat16 && t.device() == q.device() &&
           t.layout() == at::kStrided && !t.is_neg();
  };
  for (const at::Tensor* t : {&q, &k, &v, &cos, &sin, (const at::Tensor*)&cache_k,
                              (const at::Tensor*)&cache_v})
    if (!bf16_here(*t)) return none();
  // torch refuses to write an inference tensor outside inference mode
  if (!c10::InferenceMode::is_enabled() && (cache_k.is_inference() || cache_v.is_inference()))
    return none();
  if (!q.is_cuda() || q.dim() != 3 || cache_k.dim() != 4 || cache_v.dim() != 4) return none();
  const int64_t B = q.size(0), T = q.size(1), Hk = cache_k.size(1), S = cache_k.size(2);
  const int64_t D = cache_k.size(3);
  if (B < 1 || T < 1 || Hk < 1 || n_heads < 1 || n_heads % Hk != 0) return none();
  if (cache_v.sizes() != cache_k.sizes() || cache_k.size(0) < B || cache_k.stride(3) != 1 ||
      cache_v.stride(3) != 1)
    return none();
  fp_attention_args a{};
  a.ldq = token_rows(q, B, T, n_heads * D);
  a.ldk = token_rows(k, B, T, Hk * D);
  a.ldv = token_rows(v, B, T, Hk * D);
  if (a.ldq < 0 || a.ldk < 0 || a.ldv < 0) return none();
  for (const at::Tensor* t : {&cos, &sin})
    if (t->dim() != 2 || t->size(0) != T || t->size(1) != D || t->stride(1) != 1) return none();
  if (q_gamma.has_value() != k_gamma.has_value()) return none();
  if (q_gamma.has_value()) {
    for (const at::Tensor* t : {&*q_gamma, &*k_gamma})
      if (!bf16_here(*t) || t->dim() != 1 || t->size(0) != D || t->stride(0) != 1) return none();
    a.q_gamma = q_gamma->data_ptr(), a.k_gamma = k_gamma->data_ptr();
  }
  int64_t keys = S;
  if (pos.has_value()) {
    if (pos->dim() != 0 || pos->scalar_type() != at::kLong || pos->device() != q.device())
      return none();
    a.pos_dev = pos->data_ptr<int64_t>();
  } else {
    if (start_pos < 0 || start_pos + T > S) return none();
    a.pos = start_pos;
    keys = start_pos + T;
  }
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr();
  a.cos = cos.data_ptr(), a.sin = sin.data_ptr();
  a.ld_cos = T > 1 ? cos.stride(0) : D, a.ld_sin = T > 1 ? sin.stride(0) : D;
  a.cache_k = cache_k.data_ptr(), a.cache_v = cache_v.data_ptr();
  // a dimension of one element may carry any stride
  const auto sd = [](const at::Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  a.k_s_b = sd(cache_k, 0), a.k_s_h = sd(cache_k, 1), a.k_s_p = S > 1 ? cache_k.stride(2) : D;
  a.v_s_b = sd(cache_v, 0), a.v_s_h = sd(cache_v, 1), a.v_s_p = S > 1 ? cache_v.stride(2) : D;
  a.B = B, a.T = T, a.n_heads = n_heads, a.n_kv_heads = Hk, a.head_dim = D, a.cache_len = S;
  a.q_eps = (float)q_eps, a.k_eps = (float)k_eps;
  const c10::DeviceGuard guard(q.device());
  const int64_t bytes = fp_attention_workspace_bytes(B, T, n_heads, Hk, D, keys);
  if (bytes <= 0) return none();
  at::Tensor y = at::empty({B, T, n_heads * D}, q.options());
  at::Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));
  a.y = y.data_ptr();
  const int st = fp_attention_bf16(&a, ws.data_ptr(), bytes, cur_stream(q));
  // sizes, strides and alignments that the kernels do not take: nothing ran
  if (st == FP_ERR_SHAPE || st == FP_ERR_STRIDE) return none();
  check_status(st, "fp_attention_bf16");
  for (at::Tensor* t : {&cache_k, &cache_v})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return y;
}

std::tuple<at::Tensor, at::Tensor> quantize_w8(const at::Tensor& w) {
  check_2d(w, "W", at::kBFloat16);
  const c10::DeviceGuard guard(w.device());
  const int64_t N = w.size(0), K = w.size(1);
  at::Tensor q = at::empty({N, K}, w.options().dtype(at::kChar));
  at::Tensor s = at::empty({N}, w.options().dtype(at::kFloat));
  check_status(fp_quantize_w8_per_row(w.data_ptr(), w.stride(0), (int8_t*)q.data_ptr(),
                                      q.stride(0), s.data_ptr<float>(), N, K, cur_stream(w)),
               "fp_quantize_w8_per_row");
  return {q, s};
}

// ---- low-bit serving ----
//
// These ops take their tensors as the Python surface gets them (any leading dimensions
// and strides) and raise its errors themselves (ValueError, TypeError): a decode step
// of small calls is bound by the host, where each tensor operation in Python costs a
// microsecond. They are registered for CPU tensors too, for the error that says so.

void value_device(const at::Tensor& t, const char* fn, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), fn, ": ", name, " is on ", t.device(),
                    "; it runs only on a HIP (ROCm) device");
}
void value_same(const at::Tensor& x, const at::Tensor& t, const char* fn, const char* xn, const char* name) {
  TORCH_CHECK_VALUE(t.device() == x.device(), fn, ": ", xn, " (", x.device(), ") and ", name, " (", t.device(),
                    ") must be on the same device");
}
// A type's name in Python.
const char* py_name(at::ScalarType t) {
  return t == at::kByte ? "uint8" : t == at::kBFloat16 ? "bfloat16" : t == at::kHalf ? "float16" :
         t == at::kFloat ? "float32" : t == at::kLong ? "int64" : c10::toString(t);
}
void type_is(const at::Tensor& t, at::ScalarType dt, const char* fn, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == dt, fn, ": ", name, " must be ", py_name(dt), ", got ",
                   py_name(t.scalar_type()));
}

// t [.., K] as a matrix of rows that do not share memory, at less than 2^26 elements: a
// view where it can be one.
at::Tensor as_rows(const at::Tensor& t, int64_t K) {
  at::Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / (K > 0 ? K : 1), K});
  if (r.is_neg()) r = r.resolve_neg();
  const int64_t l = r.size(0) > 1 ? r.stride(0) : K;
  if ((K > 1 && r.stride(1) != 1) || l < K || l >= (int64_t)1 << 26) r = r.contiguous();
  return r;
}
// Row stride of a matrix (a single row may carry any).
int64_t ld(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// t's shape with another last dimension.
std::vector<int64_t> with_last(const at::Tensor& t, int64_t n) {
  std::vector<int64_t> s(t.sizes().begin(), t.sizes().end());
  s.back() = n;
  return s;
}

// ---- 4-bit weights ----

// Codes q [N, ceil(K/2)] and scales s [N, ceil(K/group)] of one weight of x's K inputs.
void check_w4(const char* fn, const at::Tensor& x, const at::Tensor& q, const at::Tensor& s, int64_t group) {
  const int64_t K = x.dim() ? x.size(-1) : 0;
  TORCH_CHECK_VALUE(group == 32 || group == 64 || group == 128, fn, ": group must be 32, 64 or 128, got ", group);
  TORCH_CHECK_VALUE(K >= 1, fn, ": x must have a last dimension of at least 1, got ", x.sizes());
  TORCH_CHECK_VALUE(q.dim() == 2 && q.size(1) == (K + 1) / 2, fn, ": q shape ", q.sizes(), " does not hold (N, ",
                    (K + 1) / 2, ") bytes of rows of ", K);
  TORCH_CHECK_VALUE(s.dim() == 2 && s.size(0) == q.size(0) && s.size(1) == (K + group - 1) / group, fn,
                    ": s shape ", s.sizes(), " != (", q.size(0), ", ", (K + group - 1) / group, ")");
  type_is(q, at::kByte, fn, "q");
  type_is(s, at::kBFloat16, fn, "s");
  type_is(x, at::kBFloat16, fn, "x");
  value_same(x, q, fn, "x", "q");
  value_same(x, s, fn, "x", "s");
  value_device(x, fn, "x");
}

// The norm weight as the kernels read it, or an undefined tensor.
at::Tensor w4_gamma(const char* fn, const at::Tensor& x, const c10::optional<at::Tensor>& gamma, double eps) {
  if (!gamma.has_value()) return {};
  TORCH_CHECK_VALUE(x.dim() >= 1, fn, ": x must have a last dimension of at least 1, got ", x.sizes());
  TORCH_CHECK_VALUE(gamma->dim() == 1 && gamma->size(0) == x.size(-1), fn, ": norm weight shape ", gamma->sizes(),
                    " != (", x.size(-1), ",)");
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < 3.0e38, fn, ": eps must be finite and >= 0, got ", eps);
  type_is(*gamma, at::kBFloat16, fn, "norm weight");
  value_same(x, *gamma, fn, "x", "norm weight");
  return as_rows(*gamma, gamma->size(0));
}

at::Tensor linear_w4(const at::Tensor& x, const c10::optional<at::Tensor>& gamma, double eps,
                     const at::Tensor& q_, const at::Tensor& s_, int64_t group) {
  const char* fn = "fused_linear_w4";
  const at::Tensor gm = w4_gamma(fn, x, gamma, eps);
  const void* g = gm.defined() ? gm.data_ptr() : nullptr;
  check_w4(fn, x, q_, s_, group);
  const int64_t K = x.size(-1), N = q_.size(0);
  const c10::DeviceGuard guard(x.device());
  const at::Tensor x2 = as_rows(x, K), q = as_rows(q_, q_.size(1)), s = as_rows(s_, s_.size(1));
  at::Tensor y = at::empty(with_last(x, N), x.options());
  const int64_t M = x2.size(0);
  if (M == 0 || N == 0) return y;
  const int64_t bytes = fp_w4_workspace_bytes(M, N, K, 0, g != nullptr);
  at::Tensor ws;
  if (bytes) ws = at::empty({bytes}, x.options().dtype(at::kByte));
  check_status(fp_linear_w4(x2.data_ptr(), ld(x2), g, (float)eps, q.data_ptr<uint8_t>(), ld(q), s.data_ptr(), ld(s),
                            group, y.data_ptr(), N, M, N, K, bytes ? ws.data_ptr() : nullptr, bytes, cur_stream(x)),
               "fp_linear_w4");
  return y;
}

at::Tensor gate_up_silu_w4(const at::Tensor& x, const c10::optional<at::Tensor>& gamma, double eps,
                           const at::Tensor& qg_, const at::Tensor& sg_, const at::Tensor& qu_,
                           const at::Tensor& su_, int64_t group) {
  const char* fn = "fused_gate_up_silu_w4";
  TORCH_CHECK_VALUE(qg_.sizes() == qu_.sizes(), fn, ": qg shape ", qg_.sizes(), " != qu shape ", qu_.sizes());
  const at::Tensor gm = w4_gamma(fn, x, gamma, eps);
  const void* g = gm.defined() ? gm.data_ptr() : nullptr;
  check_w4(fn, x, qg_, sg_, group);
  check_w4(fn, x, qu_, su_, group);
  const int64_t K = x.size(-1), N = qg_.size(0);
  const c10::DeviceGuard guard(x.device());
  const at::Tensor x2 = as_rows(x, K), qg = as_rows(qg_, qg_.size(1)), sg = as_rows(sg_, sg_.size(1)),
                   qu = as_rows(qu_, qu_.size(1)), su = as_rows(su_, su_.size(1));
  at::Tensor y = at::empty(with_last(x, N), x.options());
  const int64_t M = x2.size(0);
  if (M == 0 || N == 0) return y;
  const int64_t bytes = fp_w4_workspace_bytes(M, N, K, 1, g != nullptr);
  at::Tensor ws;
  if (bytes) ws = at::empty({bytes}, x.options().dtype(at::kByte));
  check_status(fp_gate_up_silu_w4(x2.data_ptr(), ld(x2), g, (float)eps, qg.data_ptr<uint8_t>(), ld(qg),
                                  sg.data_ptr(), ld(sg), qu.data_ptr<uint8_t>(), ld(qu), su.data_ptr(), ld(su),
                                  group, y.data_ptr(), N, M, N, K, bytes ? ws.data_ptr() : nullptr, bytes,
                                  cur_stream(x)),
               "fp_gate_up_silu_w4");
  return y;
}

std::tuple<at::Tensor, at::Tensor> quantize_w4(const at::Tensor& w_, int64_t group) {
  const char* fn = "quantize_w4";
  TORCH_CHECK_VALUE(w_.dim() == 2, "W must be 2D (N, K), got shape ", w_.sizes());
  TORCH_CHECK_VALUE(w_.size(1) >= 1, fn, ": rows of at least one input are taken, got shape ", w_.sizes());
  TORCH_CHECK_VALUE(group == 32 || group == 64 || group == 128, fn, ": group must be 32, 64 or 128, got ", group);
  type_is(w_, at::kBFloat16, fn, "W");
  value_device(w_, fn, "W");
  const c10::DeviceGuard guard(w_.device());
  const int64_t N = w_.size(0), K = w_.size(1);
  const at::Tensor w = as_rows(w_, K);
  at::Tensor q = at::empty({N, (K + 1) / 2}, w.options().dtype(at::kByte));
  at::Tensor s = at::empty({N, (K + group - 1) / group}, w.options());
  if (N == 0) return {q, s};
  check_status(fp_quantize_w4(w.data_ptr(), ld(w), q.data_ptr<uint8_t>(), q.size(1), s.data_ptr(), s.size(1), N, K,
                              group, cur_stream(w)),
               "fp_quantize_w4");
  return {q, s};
}

// ---- 8-bit cache ----

// A layer's cache in one buffer: the offsets of its seven parts, each 256-byte aligned.
struct Kv8Parts {
  int64_t at[7], bytes;
};
Kv8Parts kv8_parts(int64_t batch, int64_t H, int64_t D, int64_t cache_len) {
  const int64_t heads = batch * H, NB = (cache_len + 63) / 64, block = 64 * D;
  const int64_t size[7] = {heads * NB * block, heads * NB * block, heads * NB * 4, heads * NB * 4,
                           heads * 4 * block,  heads * 4 * block,  heads * 8};
  Kv8Parts p{};
  for (int i = 0; i < 7; ++i) p.at[i] = p.bytes, p.bytes += (size[i] + 255) / 256 * 256;
  return p;
}

// Where a call's buffer and tokens are: the cache's sizes {batch, heads, D, length}, pos
// (0-D or [B]) or start_pos, and lengths [B].
fp_kv8_args kv8_call(const char* fn, const at::Tensor& cache, at::IntArrayRef size, int64_t B, int64_t T,
                     int64_t start_pos, const c10::optional<at::Tensor>& pos,
                     const c10::optional<at::Tensor>& lengths) {
  TORCH_CHECK(size.size() == 4, "the sizes of an 8-bit cache are {batch, heads, D, length}");
  const Kv8Parts p = kv8_parts(size[0], size[1], size[2], size[3]);
  TORCH_CHECK(cache.scalar_type() == at::kByte && cache.dim() == 1 && cache.is_contiguous() && cache.size(0) == p.bytes,
              "the buffer of an 8-bit cache of these sizes has ", p.bytes, " contiguous bytes, got ", cache.sizes());
  TORCH_CHECK_VALUE(B <= size[0], fn, ": ", B, " sequences, the cache holds ", size[0]);
  const auto place = [&](const at::Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kLong && (t.dim() == 0 || (t.dim() == 1 && t.size(0) == B)), fn, ": ",
                      name, " must be an int64 tensor of ", B, " elements, got ", py_name(t.scalar_type()), " ",
                      t.sizes());
    TORCH_CHECK_VALUE(t.device() == cache.device() && t.is_contiguous(), fn, ": ", name, " must be contiguous on ",
                      cache.device());
  };
  fp_kv8_args a{};
  if (pos.has_value()) {
    place(*pos, "start_pos");
    a.pos_dev = pos->data_ptr<int64_t>();
    a.pos_stride = pos->dim();
  } else {
    TORCH_CHECK_VALUE(start_pos >= 0 && start_pos <= size[3] - T, fn, ": positions ", start_pos, " .. ",
                      start_pos + T - 1, " are outside the cache of ", size[3]);
    a.pos = start_pos;
  }
  if (lengths.has_value()) {
    place(*lengths, "lengths");
    TORCH_CHECK_VALUE(lengths->dim() == 1, fn, ": lengths must be an int64 tensor of ", B, " elements");
    a.lengths = lengths->data_ptr<int64_t>();
  }
  value_device(cache, fn, "the cache");
  char* base = (char*)cache.data_ptr();
  a.k_codes = (int8_t*)(base + p.at[0]), a.v_codes = (int8_t*)(base + p.at[1]);
  a.k_scale = (float*)(base + p.at[2]), a.v_scale = (float*)(base + p.at[3]);
  a.k_tail = base + p.at[4], a.v_tail = base + p.at[5], a.tail_block = (int32_t*)(base + p.at[6]);
  a.B = B, a.T = T, a.n_kv_heads = size[1], a.head_dim = size[2], a.cache_len = size[3];
  return a;
}

// t [B, T, H, D] (or [B, T, H * D]) as rows b * T + t of H * D elements at a stride that
// the kernels take: a view, or a copy.
at::Tensor kv8_rows(const at::Tensor& t, int64_t n, int64_t* ldt) {
  const int64_t B = t.size(0), T = t.size(1);
  const bool heads = t.dim() == 4;
  const bool inner = t.stride(-1) == 1 && (!heads || t.size(2) == 1 || t.stride(2) == t.size(3));
  const int64_t l = T > 1 ? t.stride(1) : B > 1 ? t.stride(0) : n;
  if (!inner || t.is_neg() || l < n || l % 4 != 0 || (B > 1 && t.stride(0) != T * l) ||
      (uintptr_t)t.data_ptr() % 8 != 0) {
    *ldt = n;
    // (clone: contiguous() leaves a tensor that is so already, at any address)
    return (t.is_neg() ? t.resolve_neg() : t).clone(at::MemoryFormat::Contiguous);
  }
  *ldt = l;
  return t;
}

void kv8_check_tokens(const char* fn, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cache,
                      at::IntArrayRef size) {
  TORCH_CHECK_VALUE(k.dim() >= 3 && k.sizes() == v.sizes() && k.numel() == k.size(0) * k.size(1) * size[1] * size[2] &&
                        (k.dim() == 3 || (k.dim() == 4 && k.size(2) == size[1])),
                    fn, ": k ", k.sizes(), " and v ", v.sizes(), " must be (B, T, ", size[1], ", ", size[2], ")");
  type_is(k, at::kBFloat16, fn, "k");
  type_is(v, at::kBFloat16, fn, "v");
  value_same(k, v, fn, "k", "v");
  value_same(k, cache, fn, "k", "the cache");
}

at::Tensor attention_kv8(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                         const c10::optional<at::Tensor>& q_gamma,
                         const c10::optional<at::Tensor>& k_gamma, double q_eps, double k_eps,
                         const c10::optional<at::Tensor>& cos, const c10::optional<at::Tensor>& sin,
                         at::Tensor cache, at::IntArrayRef size, int64_t start_pos,
                         const c10::optional<at::Tensor>& pos,
                         const c10::optional<at::Tensor>& lengths) {
  const char* fn = "attention_kv8";
  kv8_check_tokens(fn, k_, v_, cache, size);
  const int64_t B = k_.size(0), T = k_.size(1), D = size[2];
  TORCH_CHECK_VALUE(q_.dim() == k_.dim() && q_.size(0) == B && q_.size(1) == T &&
                        (q_.dim() == 3 ? q_.size(2) % D == 0 : q_.size(3) == D),
                    fn, ": q ", q_.sizes(), " must be (", B, ", ", T, ", heads, ", D, ")");
  const int64_t n = q_.dim() == 3 ? q_.size(2) : q_.size(2) * D, H = n / D;
  TORCH_CHECK_VALUE(H >= 1 && H % size[1] == 0, fn, ": ", H, " query heads are no multiple of ", size[1], " kv heads");
  type_is(q_, at::kBFloat16, fn, "q");
  value_same(k_, q_, fn, "k", "q");
  fp_kv8_args a = kv8_call(fn, cache, size, B, T, start_pos, pos, lengths);
  const c10::DeviceGuard guard(q_.device());
  at::Tensor y = at::empty(q_.sizes(), q_.options());
  if (B == 0 || T == 0) return y;
  const at::Tensor q = kv8_rows(q_, n, &a.ldq), k = kv8_rows(k_, size[1] * D, &a.ldk),
                   v = kv8_rows(v_, size[1] * D, &a.ldv);
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr(), a.n_heads = H;
  if (cos.has_value()) {
    const auto row = [&](const c10::optional<at::Tensor>& t, bool table, const char* name) -> const void* {
      if (!t.has_value()) return nullptr;
      TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->device() == q.device() && !t->is_neg() &&
                      (table ? t->dim() == 2 && t->size(0) == T && t->size(1) == D : t->dim() == 1 && t->size(0) == D) &&
                      t->stride(-1) == 1,
                  name, " has the wrong type, device, shape or stride");
      return t->data_ptr();
    };
    a.q_gamma = row(q_gamma, false, "q_gamma"), a.k_gamma = row(k_gamma, false, "k_gamma");
    a.cos = row(cos, true, "cos"), a.sin = row(sin, true, "sin");
    a.ld_cos = T > 1 ? cos->stride(0) : D;
    a.ld_sin = sin.has_value() && T > 1 ? sin->stride(0) : D;
    a.q_eps = (float)q_eps, a.k_eps = (float)k_eps;
  }
  const int64_t keys = a.pos_dev ? a.cache_len : start_pos + T;
  const int64_t bytes = fp_kv8_workspace_bytes(B, T, H, size[1], D, keys, a.cos != nullptr);
  at::Tensor ws;
  if (bytes) ws = at::empty({bytes}, q.options().dtype(at::kByte));
  a.y = y.data_ptr();
  check_status(fp_kv8_attention(&a, bytes ? ws.data_ptr() : nullptr, bytes, cur_stream(q)), "fp_kv8_attention");
  return y;
}

void write_kv8(const at::Tensor& k_, const at::Tensor& v_, at::Tensor cache, at::IntArrayRef size, int64_t start_pos,
               const c10::optional<at::Tensor>& pos, const c10::optional<at::Tensor>& lengths) {
  const char* fn = "KVCache8.write";
  kv8_check_tokens(fn, k_, v_, cache, size);
  fp_kv8_args a = kv8_call(fn, cache, size, k_.size(0), k_.size(1), start_pos, pos, lengths);
  if (a.B == 0 || a.T == 0) return;
  const c10::DeviceGuard guard(k_.device());
  const at::Tensor k = kv8_rows(k_, size[1] * size[2], &a.ldk), v = kv8_rows(v_, size[1] * size[2], &a.ldv);
  a.k = k.data_ptr(), a.v = v.data_ptr();
  check_status(fp_kv8_write(&a, cur_stream(k)), fn);
}

std::tuple<at::Tensor, at::Tensor> read_kv8(const at::Tensor& cache, at::IntArrayRef size, int64_t B, int64_t T,
                                            int64_t start_pos, const c10::optional<at::Tensor>& pos) {
  const char* fn = "KVCache8.read";
  TORCH_CHECK_VALUE(B >= 1 && T >= 1, fn, ": batch ", B, " and T ", T, " must be at least 1");
  fp_kv8_args a = kv8_call(fn, cache, size, B, T, start_pos, pos, c10::nullopt);
  const c10::DeviceGuard guard(cache.device());
  const at::TensorOptions f = cache.options().dtype(at::kFloat);
  at::Tensor k = at::empty({B, T, size[1], size[2]}, f), v = at::empty({B, T, size[1], size[2]}, f);
  check_status(fp_kv8_read(&a, k.data_ptr<float>(), v.data_ptr<float>(), cur_stream(cache)), fn);
  return {k, v};
}

std::vector<int64_t> kv8_layout(int64_t batch, int64_t H, int64_t D, int64_t cache_len) {
  const Kv8Parts p = kv8_parts(batch, H, D, cache_len);
  std::vector<int64_t> v(p.at, p.at + 7);
  v.push_back(p.bytes);
  return v;
}

// ---- log-probabilities of tokens ----

// x [.., V], tokens [..]: {logprob [..], entropy [..], top_ids [.., k], top_logprobs [.., k]}.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs(
    const at::Tensor& x_, const at::Tensor& tokens, int64_t top_k) {
  const char* fn = "token_logprobs";
  TORCH_CHECK_VALUE(x_.dim() >= 1 && tokens.sizes() == x_.sizes().slice(0, x_.dim() - 1), fn, ": tokens shape ",
                    tokens.sizes(), " != logits shape ", x_.sizes(), " without its last dim");
  const at::ScalarType dt = x_.scalar_type();
  TORCH_CHECK_TYPE(dt == at::kBFloat16 || dt == at::kHalf || dt == at::kFloat, fn,
                   ": logits must be bfloat16, float16 or float32, got ", py_name(dt));
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong, fn, ": tokens must be int64, got ",
                   py_name(tokens.scalar_type()));
  const int64_t V = x_.size(-1), most = V < 64 ? V : 64;
  TORCH_CHECK_VALUE(V >= 1 && V <= (int64_t)1 << 20, fn, ": rows of 1 to ", 1 << 20, " logits are taken, got ", V);
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= most, fn, ": top_k must be 0 to ", most, ", got ", top_k);
  value_device(x_, fn, "logits");
  value_same(x_, tokens, fn, "logits", "tokens");
  const c10::DeviceGuard guard(x_.device());
  const at::Tensor x = as_rows(x_, V), t = tokens.contiguous();
  const int64_t M = x.size(0);
  const at::TensorOptions f = x.options().dtype(at::kFloat), i = x.options().dtype(at::kLong);
  const std::vector<int64_t> top_size = with_last(x_, top_k);
  at::Tensor lp = at::empty(tokens.sizes(), f), h = at::empty(tokens.sizes(), f);
  at::Tensor ids = at::empty(top_size, i), top = at::empty(top_size, f);
  if (M == 0) return {lp, h, ids, top};
  const int64_t bytes = fp_logprob_workspace_bytes(M, V, top_k);
  at::Tensor ws;
  if (bytes) ws = at::empty({bytes}, x.options().dtype(at::kByte));
  const int dtype = dt == at::kBFloat16 ? FP_BF16 : dt == at::kHalf ? FP_F16 : FP_F32;
  check_status(fp_token_logprobs(x.data_ptr(), dtype, ld(x), t.data_ptr<int64_t>(), lp.data_ptr<float>(),
                                 h.data_ptr<float>(), ids.data_ptr<int64_t>(), top.data_ptr<float>(), M, V, top_k,
                                 bytes ? ws.data_ptr() : nullptr, bytes, cur_stream(x)),
               "fp_token_logprobs");
  return {lp, h, ids, top};
}

void low_bit(torch::Library& m) {
  m.impl("linear_w4", linear_w4);
  m.impl("gate_up_silu_w4", gate_up_silu_w4);
  m.impl("quantize_w4", quantize_w4);
  m.impl("attention_kv8", attention_kv8);
  m.impl("write_kv8", write_kv8);
  m.impl("read_kv8", read_kv8);
  m.impl("token_logprobs", token_logprobs);
}

}  // namespace

TORCH_LIBRARY(llms_amd, m) {
  m.def("qkv(Tensor x, Tensor w_qkv, int n_q, int n_k) -> Tensor");
  m.def("gate_up_silu(Tensor x, Tensor wg, Tensor wu) -> Tensor");
  m.def("qkv_w8(Tensor x, Tensor q, Tensor scale, int n_q, int n_k) -> Tensor");
  m.def("gate_up_silu_w8(Tensor x, Tensor qg, Tensor sg, Tensor qu, Tensor su) -> Tensor");
  m.def("linear(Tensor x, Tensor w) -> Tensor");
  m.def("linear_w8(Tensor x, Tensor q, Tensor scale) -> Tensor");
  m.def("rmsnorm_qkv(Tensor x, Tensor gamma, float eps, Tensor w, int n_q, int n_k) -> Tensor");
  m.def("rmsnorm_gate_up_silu(Tensor x, Tensor gamma, float eps, Tensor wg, Tensor wu) -> Tensor");
  m.def("rmsnorm_qkv_w8(Tensor x, Tensor gamma, float eps, Tensor q, Tensor scale, int n_q, "
        "int n_k) -> Tensor");
  m.def("rmsnorm_gate_up_silu_w8(Tensor x, Tensor gamma, float eps, Tensor qg, Tensor sg, "
        "Tensor qu, Tensor su) -> Tensor");
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? q_gamma, Tensor? k_gamma, float q_eps, "
        "float k_eps, Tensor cos, Tensor sin, Tensor(a!) cache_k, Tensor(b!) cache_v, "
        "int n_heads, int start_pos, Tensor? pos) -> Tensor");
  m.def("attention_kv8(Tensor q, Tensor k, Tensor v, Tensor? q_gamma, Tensor? k_gamma, float q_eps, "
        "float k_eps, Tensor? cos, Tensor? sin, Tensor(a!) cache, int[] size, int start_pos, "
        "Tensor? pos, Tensor? lengths) -> Tensor");
  m.def("write_kv8(Tensor k, Tensor v, Tensor(a!) cache, int[] size, int start_pos, Tensor? pos, "
        "Tensor? lengths) -> ()");
  m.def("read_kv8(Tensor cache, int[] size, int B, int T, int start_pos, Tensor? pos) -> "
        "(Tensor, Tensor)");
  m.def("kv8_layout(int batch, int heads, int D, int cache_len) -> int[]", kv8_layout);
  m.def("linear_w4(Tensor x, Tensor? gamma, float eps, Tensor q, Tensor scale, int group) -> Tensor");
  m.def("gate_up_silu_w4(Tensor x, Tensor? gamma, float eps, Tensor qg, Tensor sg, Tensor qu, "
        "Tensor su, int group) -> Tensor");
  m.def("quantize_w4(Tensor w, int group) -> (Tensor, Tensor)");
  m.def("token_logprobs(Tensor logits, Tensor tokens, int top_k) -> (Tensor, Tensor, Tensor, "
        "Tensor)");
  m.def("quantize_w8(Tensor w) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(llms_amd, CUDA, m) {
  m.impl("qkv", qkv);
  m.impl("gate_up_silu", gate_up_silu);
  m.impl("qkv_w8", qkv_w8);
  m.impl("gate_up_silu_w8", gate_up_silu_w8);
  m.impl("linear", linear);
  m.impl("linear_w8", linear_w8);
  m.impl("rmsnorm_qkv", rmsnorm_qkv);
  m.impl("rmsnorm_gate_up_silu", rmsnorm_gate_up_silu);
  m.impl("rmsnorm_qkv_w8", rmsnorm_qkv_w8);
  m.impl("rmsnorm_gate_up_silu_w8", rmsnorm_gate_up_silu_w8);
  m.impl("attention", attention);
  m.impl("quantize_w8", quantize_w8);
  low_bit(m);
}

TORCH_LIBRARY_IMPL(llms_amd, CPU, m) { low_bit(m); }
