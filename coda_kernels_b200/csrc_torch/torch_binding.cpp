// Compiled dispatch layer: the device operators of the four fused-linear functions registered with PyTorch from C++
// (TORCH_LIBRARY, namespace coda_b200n), each a thin call into the C ABI of libcoda_b200.so.  It does what the ctypes
// table in _lib.py does, without the per-launch Python work: tensors in, pointers / strides / extents / the current
// CUDA stream out.  The `*_out` ops allocate nothing: they mutate the outputs the Python wrapper passes in and return
// nothing, the convention of the reference's `_kernel_op` (coda/core/gemm/gemm_interface.py:78-100).  Below them sit
// whole-operator entry points (`swiglu_fwd`, `swiglu_bwd`, ...): one dispatcher call per direction of an autograd node,
// which allocates the outputs with the caching allocator and issues that direction's launches back to back, so a short
// step (a head-sharded rank, a small batch) is not bound by the interpreter between launches.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <climits>
#include <cmath>
#include <initializer_list>
#include <tuple>

#include "../../include/coda_b200.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

inline void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", coda_b200_last_error());
}
inline void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
inline int* status_ptr(const Tensor& status) { return status.data_ptr<int>(); }
inline const void* ptr_or_null(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

void gemm_out(const Tensor& A, const Tensor& B, Tensor& out, const OptTensor& alpha, const OptTensor& C, const Tensor& status) {
  const c10::cuda::CUDAGuard guard(A.device());
  const int M = static_cast<int>(A.size(0)), N = static_cast<int>(B.size(1)), K = static_cast<int>(A.size(1));
  const float* alpha_ptr = alpha.has_value() ? alpha->data_ptr<float>() : nullptr;
  if (!C.has_value()) {
    // A plain product may be balanced by stream-K; its fp32 workspace (the one allocation of this layer's `*_out` ops)
    // comes from the caching allocator and is only asked for when the library would use it.
    const int64_t ws_bytes = coda_b200_gemm_workspace_bytes(M, N, K);
    Tensor ws;
    if (ws_bytes > 0) ws = at::empty({ws_bytes / 4}, A.options().dtype(at::kFloat));
    check(coda_b200_gemm_ws(A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0), B.stride(1), out.data_ptr(), out.stride(0),
                            out.scalar_type() == at::kFloat, M, N, K, alpha_ptr, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
                            status_ptr(status), stream_of(A)),
          "gemm");
    return;
  }
  check(coda_b200_gemm_add(A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0), B.stride(1), C->data_ptr(), C->stride(0),
                           C->scalar_type() == at::kFloat, out.data_ptr(), out.stride(0), out.scalar_type() == at::kFloat, M, N, K,
                           alpha_ptr, status_ptr(status), stream_of(A)),
        "gemm");
}

void gemm_sigmoid_out(const Tensor& A, const Tensor& B, Tensor& out, const Tensor& status) {
  const c10::cuda::CUDAGuard guard(A.device());
  check(coda_b200_gemm_sigmoid(A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0), B.stride(1), out.data_ptr(),
                               out.stride(0), out.scalar_type() == at::kFloat, static_cast<int>(A.size(0)), static_cast<int>(B.size(1)),
                               static_cast<int>(A.size(1)), status_ptr(status), stream_of(A)),
        "gemm_sigmoid");
}

void gemm_swiglu_out(const Tensor& A, const Tensor& B, Tensor& preact, Tensor& postact, const Tensor& status) {
  const c10::cuda::CUDAGuard guard(A.device());
  check(coda_b200_gemm_swiglu(A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0), B.stride(1), preact.data_ptr(),
                              preact.stride(0), postact.data_ptr(), postact.stride(0), static_cast<int>(A.size(0)),
                              static_cast<int>(B.size(1)), static_cast<int>(A.size(1)), status_ptr(status), stream_of(A)),
        "gemm_swiglu");
}

void gemm_lse_out(const Tensor& A, const Tensor& B, const OptTensor& probs, Tensor& part_max, Tensor& part_sum, const Tensor& target,
                  Tensor& target_logit, const Tensor& status) {
  const c10::cuda::CUDAGuard guard(A.device());
  check(coda_b200_gemm_lse(A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0), B.stride(1),
                           probs.has_value() ? probs->data_ptr() : nullptr, probs.has_value() ? probs->stride(0) : 0,
                           part_max.data_ptr<float>(), part_sum.data_ptr<float>(), target.data_ptr<int32_t>(),
                           target_logit.data_ptr<float>(), static_cast<int>(A.size(0)), static_cast<int>(B.size(1)),
                           static_cast<int>(A.size(1)), status_ptr(status), stream_of(A)),
        "gemm_lse");
}

void lse_finalize_out(const Tensor& part_max, const Tensor& part_sum, const Tensor& target, const Tensor& target_logit,
                      int64_t ignore_index, Tensor& lse, Tensor& losses) {
  const c10::cuda::CUDAGuard guard(part_max.device());
  check(coda_b200_lse_finalize(part_max.data_ptr<float>(), part_sum.data_ptr<float>(), static_cast<int>(part_max.size(1)),
                               target.data_ptr<int32_t>(), target_logit.data_ptr<float>(), static_cast<int>(ignore_index),
                               lse.data_ptr<float>(), losses.data_ptr<float>(), static_cast<int>(part_max.size(0)), stream_of(part_max)),
        "lse_finalize");
}

void ce_grad_fixup_(Tensor& probs, const Tensor& part_max, const Tensor& lse, const Tensor& target, int64_t ignore_index) {
  const c10::cuda::CUDAGuard guard(probs.device());
  check(coda_b200_ce_grad_fixup(probs.data_ptr(), probs.stride(0), part_max.data_ptr<float>(), static_cast<int>(part_max.size(1)),
                                lse.data_ptr<float>(), target.data_ptr<int32_t>(), static_cast<int>(ignore_index),
                                static_cast<int>(probs.size(0)), static_cast<int>(probs.size(1)), stream_of(probs)),
        "ce_grad_fixup");
}

void gemm_qknorm_rope_out(const Tensor& A, const Tensor& B, Tensor& qk, Tensor& preact, const OptTensor& v, Tensor& mean_sq,
                          const Tensor& gamma, const Tensor& positions, const Tensor& frequencies, int64_t head_dim, int64_t hq,
                          int64_t hk, double eps, const Tensor& status) {
  const c10::cuda::CUDAGuard guard(A.device());
  check(coda_b200_gemm_qknorm_rope(A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0), B.stride(1), qk.data_ptr(),
                                   qk.stride(0), preact.data_ptr(), preact.stride(0), v.has_value() ? v->data_ptr() : nullptr,
                                   v.has_value() ? v->stride(0) : 0, mean_sq.data_ptr<float>(), gamma.data_ptr(), positions.data_ptr(),
                                   positions.scalar_type() == at::kFloat, frequencies.data_ptr<float>(), static_cast<int>(head_dim),
                                   static_cast<int>(hq), static_cast<int>(hk), static_cast<float>(eps), static_cast<int>(A.size(0)),
                                   static_cast<int>(B.size(1)), static_cast<int>(A.size(1)), status_ptr(status), stream_of(A)),
        "gemm_qknorm_rope");
}

void dswiglu_out(const Tensor& preact, const Tensor& dout, Tensor& grad_pre) {
  const c10::cuda::CUDAGuard guard(dout.device());
  check(coda_b200_dswiglu(preact.data_ptr(), preact.stride(0), dout.data_ptr(), dout.stride(0), grad_pre.data_ptr(), grad_pre.stride(0),
                          static_cast<int>(dout.size(0)), static_cast<int>(dout.size(1)), stream_of(dout)),
        "dswiglu");
}

void dsigmoid_out(const Tensor& out, const Tensor& dout, Tensor& grad_pre) {
  const c10::cuda::CUDAGuard guard(dout.device());
  check(coda_b200_dsigmoid(out.data_ptr(), out.stride(0), out.scalar_type() == at::kFloat, dout.data_ptr(), dout.stride(0),
                           grad_pre.data_ptr(), grad_pre.stride(0), static_cast<int>(dout.size(0)), static_cast<int>(dout.size(1)),
                           stream_of(dout)),
        "dsigmoid");
}

void qknorm_rope_bwd_out(const Tensor& dq, const Tensor& dk, const OptTensor& dv, const Tensor& preact, const Tensor& mean_sq,
                         const Tensor& gamma, const Tensor& positions, const Tensor& frequencies, int64_t head_dim, int64_t hq, int64_t hk,
                         double eps, Tensor& grad, Tensor& dgamma, Tensor& scratch) {
  const c10::cuda::CUDAGuard guard(preact.device());
  check(coda_b200_qknorm_rope_bwd(dq.data_ptr(), dq.stride(0), dk.data_ptr(), dk.stride(0), dv.has_value() ? dv->data_ptr() : nullptr,
                                  dv.has_value() ? dv->stride(0) : 0, dv.has_value() ? static_cast<int>(dv->size(1)) : 0, preact.data_ptr(),
                                  preact.stride(0), mean_sq.data_ptr<float>(), gamma.data_ptr(), positions.data_ptr(),
                                  positions.scalar_type() == at::kFloat, frequencies.data_ptr<float>(), static_cast<int>(head_dim),
                                  static_cast<int>(hq), static_cast<int>(hk), static_cast<float>(eps), grad.data_ptr(), grad.stride(0),
                                  dgamma.data_ptr<float>(), scratch.data_ptr(), static_cast<int64_t>(scratch.numel() * scratch.element_size()),
                                  static_cast<int>(preact.size(0)), stream_of(preact)),
        "qknorm_rope_bwd");
}

// ---------------------------------------------------------------------------------------- whole-operator entry points

using OptPair = std::tuple<OptTensor, OptTensor>;

inline void require_bf16(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2, name, " must be a 2-D bfloat16 CUDA tensor");
}
inline Tensor new_matrix(const Tensor& like, int64_t rows, int64_t cols, at::ScalarType dtype) {
  return at::empty({rows, cols}, like.options().dtype(dtype));
}
// Contiguous and 16-byte aligned: gamma and the rotary frequencies are read 16 bytes at a time.
inline Tensor aligned16(const Tensor& t) {
  Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0 ? c : c.clone();
}

// dx = alpha * grad_pre @ weight, dweight = alpha * grad_pre^T @ x (either may be skipped).  The [N, K] weight and
// both operands of the weight gradient are consumed as MN-major views: no transposed copy.
OptPair linear_backward(const Tensor& grad_pre, const Tensor& x, const Tensor& weight, bool need_dx, bool need_dw, const OptTensor& alpha,
                        const Tensor& status) {
  require_bf16(grad_pre, "grad_pre");
  require_bf16(x, "x");
  require_bf16(weight, "weight");
  OptTensor dx, dw;
  if (need_dx) {
    Tensor out = new_matrix(x, grad_pre.size(0), weight.size(1), at::kBFloat16);
    gemm_out(grad_pre, weight, out, alpha, c10::nullopt, status);
    dx = out;
  }
  if (need_dw) {
    Tensor out = new_matrix(x, grad_pre.size(1), x.size(1), at::kBFloat16);
    gemm_out(grad_pre.t(), x, out, alpha, c10::nullopt, status);
    dw = out;
  }
  return {dx, dw};
}

std::tuple<Tensor, Tensor> swiglu_fwd(const Tensor& x, const Tensor& weight, const Tensor& status) {
  require_bf16(x, "x");
  require_bf16(weight, "weight");
  TORCH_CHECK(weight.size(0) % 2 == 0, "gemm_swiglu: N must be even");
  Tensor preact = new_matrix(x, x.size(0), weight.size(0), at::kBFloat16);
  Tensor postact = new_matrix(x, x.size(0), weight.size(0) / 2, at::kBFloat16);
  gemm_swiglu_out(x, weight.t(), preact, postact, status);
  return {preact, postact};
}

OptPair swiglu_bwd(const Tensor& preact, const Tensor& dout, const Tensor& x, const Tensor& weight, bool need_dx, bool need_dw,
                   const Tensor& status) {
  require_bf16(preact, "preact");
  require_bf16(dout, "dout");
  TORCH_CHECK(preact.stride(1) == 1 && dout.stride(1) == 1 && preact.size(1) == 2 * dout.size(1) && preact.size(0) == dout.size(0),
              "dswiglu: bad shapes");
  Tensor grad_pre = at::empty_like(preact);
  dswiglu_out(preact, dout, grad_pre);
  return linear_backward(grad_pre, x, weight, need_dx, need_dw, c10::nullopt, status);
}

Tensor sigmoid_fwd(const Tensor& x, const Tensor& weight, bool out_fp32, const Tensor& status) {
  require_bf16(x, "x");
  require_bf16(weight, "weight");
  Tensor out = new_matrix(x, x.size(0), weight.size(0), out_fp32 ? at::kFloat : at::kBFloat16);
  gemm_sigmoid_out(x, weight.t(), out, status);
  return out;
}

OptPair sigmoid_bwd(const Tensor& out, const Tensor& dout, const Tensor& x, const Tensor& weight, bool need_dx, bool need_dw,
                    const Tensor& status) {
  require_bf16(dout, "dout");
  TORCH_CHECK(out.sizes() == dout.sizes() && (out.scalar_type() == at::kBFloat16 || out.scalar_type() == at::kFloat), "dsigmoid: bad out");
  Tensor grad_pre = at::empty_like(dout);
  dsigmoid_out(out, dout, grad_pre);
  return linear_backward(grad_pre, x, weight, need_dx, need_dw, c10::nullopt, status);
}

// (loss, 1 / count or nothing, gradient of the summed row losses w.r.t. the logits or nothing).  With `store_grad` the
// [M, V] buffer first receives unnormalised probabilities from the GEMM epilogue and is then rewritten in place to
// softmax - onehot; without it nothing of that size exists.
std::tuple<Tensor, OptTensor, OptTensor> cross_entropy_fwd(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t ignore_index,
                                                           bool mean, bool store_grad, const Tensor& status) {
  require_bf16(x, "x");
  require_bf16(weight, "weight");
  TORCH_CHECK(target.is_cuda() && target.scalar_type() == at::kInt && target.is_contiguous() && target.numel() == x.size(0),
              "target must be a contiguous int32 CUDA tensor with one label per row");
  const int64_t M = x.size(0), V = weight.size(0);
  const int64_t tiles = coda_b200_lse_tiles(static_cast<int>(V));
  const auto f32 = x.options().dtype(at::kFloat);
  OptTensor probs;
  if (store_grad) probs = new_matrix(x, M, V, at::kBFloat16);
  Tensor part_max = at::empty({M, tiles}, f32), part_sum = at::empty({M, tiles}, f32);
  Tensor target_logit = at::zeros({M}, f32), lse = at::empty({M}, f32), losses = at::empty({M}, f32);
  gemm_lse_out(x, weight.t(), probs, part_max, part_sum, target, target_logit, status);
  lse_finalize_out(part_max, part_sum, target, target_logit, ignore_index, lse, losses);
  if (store_grad) ce_grad_fixup_(*probs, part_max, lse, target, ignore_index);
  Tensor loss = losses.sum();
  OptTensor inv_count;
  if (mean) {  // ignored rows already carry an exact zero; the divisor stays on the device
    inv_count = target.ne(ignore_index).sum().to(at::kFloat).reciprocal();
    loss = loss * *inv_count;
  }
  return {loss, inv_count, probs};
}

OptPair cross_entropy_bwd(const Tensor& dloss, const OptTensor& inv_count, const Tensor& dlogits, const Tensor& x, const Tensor& weight,
                          bool need_dx, bool need_dw, const Tensor& status) {
  const Tensor alpha = (inv_count.has_value() ? dloss * *inv_count : dloss).reshape({1}).to(at::kFloat);
  return linear_backward(dlogits, x, weight, need_dx, need_dw, alpha, status);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qknorm_rope_fwd(const Tensor& x, const Tensor& weight, const Tensor& gamma, const Tensor& positions,
                                                          const Tensor& frequencies, int64_t head_dim, int64_t hq, int64_t hk, double eps,
                                                          const Tensor& status) {
  require_bf16(x, "x");
  require_bf16(weight, "weight");
  TORCH_CHECK(gamma.is_cuda() && gamma.scalar_type() == at::kBFloat16 && gamma.numel() == 2 * head_dim, "gamma must hold [gamma_q | gamma_k]");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kFloat, "positions must be int32 or float32");
  TORCH_CHECK(frequencies.scalar_type() == at::kFloat, "frequencies must be float32");
  const int64_t M = x.size(0), N = weight.size(0), heads = hq + hk, size_qk = heads * head_dim;
  TORCH_CHECK(frequencies.numel() == size_qk, "frequencies must have (hq + hk) * head_dim entries");
  TORCH_CHECK(positions.numel() == M, "positions must have one entry per row");
  TORCH_CHECK(N >= size_qk, "weight has fewer rows than the q and k heads need");
  Tensor qk = new_matrix(x, M, size_qk, at::kBFloat16), preact = new_matrix(x, M, size_qk, at::kBFloat16);
  Tensor mean_sq = new_matrix(x, M, heads, at::kFloat), v = new_matrix(x, M, N - size_qk, at::kBFloat16);
  OptTensor v_arg;
  if (N > size_qk) v_arg = v;
  gemm_qknorm_rope_out(x, weight.t(), qk, preact, v_arg, mean_sq, aligned16(gamma), positions.contiguous(), aligned16(frequencies), head_dim,
                       hq, hk, eps, status);
  return {qk, preact, mean_sq, v};
}

// (dx, dweight, dgamma in gamma's dtype).  [grad_pre | dv] is one buffer, so each GEMM of the backward runs once over
// the whole [q | k | v] weight.
std::tuple<OptTensor, OptTensor, Tensor> qknorm_rope_bwd(const Tensor& dq, const Tensor& dk, const Tensor& dv, const Tensor& x,
                                                         const Tensor& weight, const Tensor& preact, const Tensor& mean_sq, const Tensor& gamma,
                                                         const Tensor& positions, const Tensor& frequencies, int64_t head_dim, int64_t hq,
                                                         int64_t hk, double eps, bool need_dx, bool need_dw, const Tensor& status) {
  require_bf16(dq, "dq");
  require_bf16(dk, "dk");
  require_bf16(preact, "preact");
  const int64_t M = preact.size(0), size_qk = preact.size(1), nv = dv.size(1);
  Tensor grad = new_matrix(x, M, size_qk + nv, at::kBFloat16);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor dgamma = at::empty({2 * head_dim}, f32);
  const int64_t scratch_bytes = coda_b200_qknorm_rope_bwd_scratch_bytes(static_cast<int>(M), static_cast<int>(head_dim));
  Tensor scratch = at::empty({(scratch_bytes + 3) / 4}, f32);
  OptTensor dv_arg;
  if (nv > 0) {
    require_bf16(dv, "dv");
    dv_arg = dv;
  }
  qknorm_rope_bwd_out(dq, dk, dv_arg, preact, mean_sq, aligned16(gamma), positions.contiguous(), aligned16(frequencies), head_dim, hq, hk,
                      eps, grad, dgamma, scratch);
  auto [dx, dw] = linear_backward(grad, x, weight, need_dx, need_dw, c10::nullopt, status);
  return {dx, dw, dgamma.to(gamma.scalar_type())};
}

// ---------------------------------------------------------------------------------------- around the fused linears
// Operators whose kernels take microseconds: the whole call, autograd node and argument checks included, is C++, in two
// layers.  The functions on the CUDA key check the arguments and launch; those on the Autograd key (namespace autograd)
// decide whether a node is needed, and they and the nodes reach the CUDA functions through the dispatcher, forward and
// backward, so that a tracer or a dispatch mode sees every computation as an operator.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline void require_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "coda_b200 operators run on CUDA tensors only; there is no CPU fallback");
}
inline void require_rows(const Tensor& x) {
  require_cuda(x);
  const auto dt = x.scalar_type();
  TORCH_CHECK_NOT_IMPLEMENTED(dt == at::kBFloat16 || dt == at::kHalf || dt == at::kFloat,
                              "coda_b200 row operators take bfloat16, float16 or float32, got ", dt);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must have a last dimension of at least one element");
}
inline void require_like(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.device() == x.device() && t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes(), name,
                    " must match x in shape, dtype and device");
}
inline void require_weight(const Tensor& w, const Tensor& x) {
  TORCH_CHECK_VALUE(w.device() == x.device() && w.scalar_type() == x.scalar_type() && w.dim() == 1 && w.size(0) == x.size(-1),
                    "weight must hold one entry per column of x, in x's dtype, on x's device");
}
inline void require_dropout(const Tensor& x, double p, const OptTensor& rng, int64_t stream) {
  TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0, "the dropout probability must be at least 0 and below 1, got ", p);
  TORCH_CHECK_VALUE(stream >= 0 && stream <= 0xffffffffLL, "the dropout stream must be a 32-bit number");
  TORCH_CHECK_VALUE(p == 0.0 || rng.has_value(), "dropout needs rng, an int64 CUDA tensor [seed, step]");
  if (rng.has_value())
    TORCH_CHECK_VALUE(rng->device() == x.device() && rng->scalar_type() == at::kLong && rng->dim() == 1 && rng->size(0) == 2,
                      "rng must be an int64 tensor [seed, step] on x's device");
}
// A tangent would be dropped without a word by the plain path: the result would read as if the derivative were zero.
inline void require_no_tangent(const char* name, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative");
}
inline void require_no_grad(const char* name, std::initializer_list<const Tensor*> tensors) {
  require_no_tangent(name, tensors);
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t->defined() || !t->requires_grad(), name, " has no backward: call it under torch.no_grad() or on detached tensors");
}
inline void require_first_order(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " can be differentiated once only");
}
inline bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->requires_grad()) return true;
  return false;
}
// An operator of this file through the dispatcher: below autograd, but seen by modes.
template <typename Signature>
c10::TypedOperatorHandle<Signature> operator_named(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}
inline OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
inline int row_dtype(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : 2;
}
inline const int64_t* rng_ptr(const Tensor& rng) { return rng.defined() ? rng.data_ptr<int64_t>() : nullptr; }
inline void* ptr_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline Tensor dense(const OptTensor& t) { return t.has_value() ? aligned16(*t) : Tensor(); }

// dropout of x from rng; `used` (when wanted) receives the [seed, step] the mask was made from
Tensor run_dropout(const Tensor& x_in, double p, const OptTensor& rng_in, int64_t stream, Tensor* used) {
  require_rows(x_in);
  require_dropout(x_in, p, rng_in, stream);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned16(x_in), rng = dense(rng_in);
  Tensor out = at::empty_like(x);
  if (used != nullptr) *used = at::empty({2}, x.options().dtype(at::kLong));
  check(coda_b200_dropout(x.data_ptr(), out.data_ptr(), x.numel() / x.size(-1), x.size(-1), row_dtype(x), p, rng_ptr(rng), stream,
                          used != nullptr ? used->data_ptr<int64_t>() : nullptr, stream_of(x)),
        "dropout");
  return out;
}
Tensor dropout(const Tensor& x, double p, const OptTensor& rng, int64_t stream) { return run_dropout(x, p, rng, stream, nullptr); }
// (out, the [seed, step] used)
std::tuple<Tensor, Tensor> dropout_fwd(const Tensor& x, double p, const OptTensor& rng, int64_t stream) {
  Tensor used, out = run_dropout(x, p, rng, stream, &used);
  return {out, used};
}

// (out, h or nothing without a residual, rstd, the [seed, step] used or nothing without dropout, and with keep_low the bits of h
// below a 2-byte type)
std::tuple<Tensor, OptTensor, Tensor, OptTensor, OptTensor> norm_fwd(const Tensor& x_in, const OptTensor& residual_in, const Tensor& weight_in,
                                                                     double eps, double p, const OptTensor& rng_in, int64_t stream,
                                                                     bool keep_low) {
  require_rows(x_in);
  if (residual_in.has_value()) require_like(*residual_in, x_in, "residual");
  require_weight(weight_in, x_in);
  require_dropout(x_in, p, rng_in, stream);
  TORCH_CHECK_VALUE(p == 0.0 || residual_in.has_value(), "dropout needs a residual");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned16(x_in), residual = dense(residual_in), weight = aligned16(weight_in), rng = dense(rng_in);
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  Tensor out = at::empty_like(x), rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  OptTensor h, used, low;
  if (residual.defined()) h = at::empty_like(x);
  if (keep_low && h.has_value() && x.element_size() == 2)
    low = at::empty({coda_b200_add_rmsnorm_low_bytes(rows, cols) / 4}, x.options().dtype(at::kInt));
  if (p > 0.0) used = at::empty({2}, x.options().dtype(at::kLong));
  auto to = [](const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; };
  check(coda_b200_add_rmsnorm_fwd_low(x.data_ptr(), ptr_or_null(residual), weight.data_ptr(), static_cast<float>(eps), p, rng_ptr(rng), stream,
                                      static_cast<int64_t*>(to(used)), to(h), to(low), out.data_ptr(), rstd.data_ptr<float>(), rows, cols,
                                      row_dtype(x), stream_of(x)),
        "add_rmsnorm");
  return {out, h, rstd, used, low};
}
// (dx, dres, dweight), nothing where not wanted; dout undefined: only h was used
std::tuple<OptTensor, OptTensor, OptTensor> norm_bwd(const OptTensor& dout_in, const OptTensor& dh_in, const Tensor& h_in,
                                                     const OptTensor& low_in, const Tensor& rstd, const Tensor& weight_in, double p,
                                                     const OptTensor& rng_in, int64_t stream, bool need_dx, bool need_dres, bool need_dw) {
  require_rows(h_in);
  if (dout_in.has_value()) require_like(*dout_in, h_in, "dout");
  if (dh_in.has_value()) require_like(*dh_in, h_in, "dh");
  require_weight(weight_in, h_in);
  require_dropout(h_in, p, rng_in, stream);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(h_in.device());
  if (low_in.has_value())
    TORCH_CHECK_VALUE(low_in->device() == h_in.device() && low_in->scalar_type() == at::kInt &&
                          4 * low_in->numel() == coda_b200_add_rmsnorm_low_bytes(h_in.numel() / h_in.size(-1), h_in.size(-1)),
                      "the bits below h must be int32, as many as the forward left");
  const Tensor h = aligned16(h_in), weight = aligned16(weight_in), rng = dense(rng_in), dh = dense(dh_in), low = dense(low_in);
  const Tensor dout = dout_in.has_value() ? aligned16(*dout_in) : at::zeros_like(h);
  const int64_t cols = h.size(-1), rows = h.numel() / cols;
  TORCH_CHECK_VALUE(rstd.device() == h.device() && rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == rows,
                    "rstd must be float32 with one entry per row");
  OptTensor dx, dres, dw;
  Tensor scratch;
  if (need_dx) dx = at::empty_like(h);
  if (need_dres) dres = at::empty_like(h);
  int64_t scratch_bytes = 0;
  if (need_dw) {
    dw = rows > 0 ? at::empty_like(weight) : at::zeros_like(weight);
    scratch_bytes = coda_b200_add_rmsnorm_bwd_scratch_bytes(rows, cols);
    scratch = at::empty({scratch_bytes / 4}, h.options().dtype(at::kFloat));
  }
  auto to = [](const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; };
  check(coda_b200_add_rmsnorm_bwd_low(dout.data_ptr(), ptr_or_null(dh), h.data_ptr(), ptr_or_null(low), rstd.data_ptr<float>(),
                                      weight.data_ptr(), p, rng_ptr(rng), stream, to(dx), to(dres), to(dw), ptr_or_null(scratch),
                                      scratch_bytes, rows, cols, row_dtype(h), stream_of(h)),
        "add_rmsnorm backward");
  return {dx, dres, dw};
}
Tensor rms_norm(const Tensor& x, const Tensor& weight, double eps) {
  return std::get<0>(norm_fwd(x, c10::nullopt, weight, eps, 0.0, c10::nullopt, 0, false));
}
std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps, double p,
                                        const OptTensor& rng, int64_t stream) {
  auto f = norm_fwd(x, residual, weight, eps, p, rng, stream, false);
  return {std::get<0>(f), *std::get<1>(f)};
}

// (q, scale, h or nothing)
std::tuple<Tensor, Tensor, OptTensor> rows_e4m3(const Tensor& x_in, const OptTensor& residual_in, const OptTensor& weight_in, double eps) {
  require_rows(x_in);
  if (residual_in.has_value()) require_like(*residual_in, x_in, "residual");
  if (weight_in.has_value()) require_weight(*weight_in, x_in);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned16(x_in), residual = dense(residual_in), weight = dense(weight_in);
  Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  OptTensor h;
  if (residual.defined()) h = at::empty_like(x);
  check(coda_b200_rows_e4m3(x.data_ptr(), ptr_or_null(residual), ptr_or_null(weight), static_cast<float>(eps),
                            h.has_value() ? h->data_ptr() : nullptr, q.data_ptr(), scale.data_ptr<float>(), x.numel() / x.size(-1), x.size(-1),
                            row_dtype(x), stream_of(x)),
        "rows_e4m3");
  return {q, scale, h};
}

Tensor linear_e4m3(const Tensor& x_in, const Tensor& x_scale, const Tensor& weight_in, const Tensor& weight_scale, bool out_fp32,
                   const Tensor& status) {
  for (const Tensor* t : {&x_in, &x_scale, &weight_in, &weight_scale}) {
    require_cuda(*t);
    TORCH_CHECK_VALUE(t->device() == x_in.device(), "all operands must be on one device");
  }
  TORCH_CHECK_NOT_IMPLEMENTED(x_in.scalar_type() == at::kFloat8_e4m3fn && weight_in.scalar_type() == at::kFloat8_e4m3fn,
                              "x and weight must be float8_e4m3fn, got ", x_in.scalar_type(), " and ", weight_in.scalar_type());
  TORCH_CHECK_VALUE(x_in.dim() == 2 && weight_in.dim() == 2 && x_in.size(1) == weight_in.size(1), "x [M, K] and weight [N, K] expected");
  const int64_t M = x_in.size(0), N = weight_in.size(0), K = x_in.size(1);
  TORCH_CHECK_VALUE(K > 0 && K % 16 == 0, "K must be a positive multiple of 16");
  TORCH_CHECK_VALUE(N > 0 && N % 8 == 0, "the number of weight rows must be a positive multiple of 8");
  TORCH_CHECK_VALUE(x_scale.scalar_type() == at::kFloat && x_scale.dim() == 1 && x_scale.size(0) == M,
                    "x_scale must be float32 with one entry per row");
  TORCH_CHECK_VALUE(weight_scale.scalar_type() == at::kFloat && weight_scale.dim() == 1 && weight_scale.size(0) == N,
                    "weight_scale must be float32 with one entry per row");
  TORCH_CHECK_VALUE(M <= INT_MAX && N <= INT_MAX && K <= INT_MAX, "extents must fit 31 bits");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned16(x_in), xs = x_scale.contiguous(), weight = aligned16(weight_in), ws = weight_scale.contiguous();
  Tensor out = new_matrix(x, M, N, out_fp32 ? at::kFloat : at::kBFloat16);
  if (M == 0) return out;
  const int64_t parts_bytes = coda_b200_gemm_e4m3_workspace_bytes(static_cast<int>(M), static_cast<int>(N), static_cast<int>(K));
  Tensor parts;
  if (parts_bytes > 0) parts = at::empty({parts_bytes / 4}, x.options().dtype(at::kFloat));
  check(coda_b200_gemm_e4m3(x.data_ptr(), xs.data_ptr<float>(), weight.data_ptr(), ws.data_ptr<float>(), out.data_ptr(), N, out_fp32,
                            static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), ptr_or_null(parts), parts_bytes, status_ptr(status),
                            stream_of(x)),
        "gemm_e4m3");
  return out;
}

// What the loss's products work on: x and target, or, where that pays, the rows that count put first (then `live` says how
// many, and `position` where each row went).  Every matrix operand is dense, so its strides are its extents.
struct CeRows {
  Tensor x, target, position, live;
};
inline bool ce_compacts(const Tensor& x, const Tensor& weight) {
  if (x.dim() != 2 || weight.dim() != 2) return false;  // (refused where the arguments are checked)
  for (const int64_t n : {x.size(0), weight.size(0), x.size(-1)})
    if (n < 1 || n > INT_MAX) return false;
  return coda_b200_ce_compacts(static_cast<int>(x.size(0)), static_cast<int>(weight.size(0)), static_cast<int>(x.size(-1))) != 0;
}
CeRows ce_rows(const Tensor& x, const Tensor& target, int64_t ignore_index, bool compact) {
  if (!compact) return {x, target, Tensor(), Tensor()};
  const int M = static_cast<int>(x.size(0)), K = static_cast<int>(x.size(1));
  CeRows r{at::empty_like(x), at::empty_like(target), at::empty_like(target), at::empty({1}, target.options())};
  check(coda_b200_ce_compact(x.data_ptr(), target.data_ptr<int32_t>(), static_cast<int>(ignore_index), r.position.data_ptr<int32_t>(),
                             r.target.data_ptr<int32_t>(), r.live.data_ptr<int32_t>(), r.x.data_ptr(), M, K, stream_of(x)),
        "ce_compact");
  return r;
}
inline const int32_t* live_ptr(const Tensor& live) { return live.defined() ? live.data_ptr<int32_t>() : nullptr; }

// (loss, inv_count, lse)
std::tuple<Tensor, Tensor, Tensor> run_ce(const CeRows& r, const Tensor& weight, int64_t ignore_index, bool mean, const Tensor& status) {
  const Tensor& x = r.x;
  const int64_t M = x.size(0), V = weight.size(0), K = x.size(1);
  const auto f32 = x.options().dtype(at::kFloat);
  if (M == 0)  // a sum over nothing, and 0 / 0
    return {at::full({}, mean ? NAN : 0.0, f32), at::zeros({}, f32), at::empty({0}, f32)};
  const int64_t tiles = coda_b200_lse_tiles(static_cast<int>(V));
  Tensor parts = at::empty({2 * M * tiles + 2 * M}, f32), lse = at::empty({M}, f32), loss = at::empty({}, f32), inv_count = at::empty({}, f32);
  float* part = parts.data_ptr<float>();
  check(coda_b200_ce_loss(x.data_ptr(), K, 1, weight.data_ptr(), 1, K, r.target.data_ptr<int32_t>(), static_cast<int>(ignore_index), mean,
                          live_ptr(r.live), part, part + M * tiles, part + 2 * M * tiles, lse.data_ptr<float>(), part + 2 * M * tiles + M,
                          loss.data_ptr<float>(), inv_count.data_ptr<float>(), static_cast<int>(M), static_cast<int>(V), static_cast<int>(K),
                          status_ptr(status), stream_of(x)),
        "ce_loss");
  return {loss, inv_count, lse};
}

// out = alpha A @ B (+ C, fp32 of out's layout) for operands of any contiguous extent
void gemm_ragged(const Tensor& A, const Tensor& B, const Tensor& out, const Tensor& alpha, const OptTensor& C, const Tensor& status) {
  const int M = static_cast<int>(A.size(0)), N = static_cast<int>(B.size(1)), K = static_cast<int>(A.size(1));
  const int64_t ws_bytes = C.has_value() ? 0 : coda_b200_gemm_workspace_bytes(M, N, K);
  Tensor ws;
  if (ws_bytes > 0) ws = at::empty({ws_bytes / 4}, alpha.options());
  check(coda_b200_gemm_ragged(A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0), B.stride(1),
                              C.has_value() ? C->data_ptr<float>() : nullptr, out.data_ptr(), out.stride(0), out.scalar_type() == at::kFloat,
                              M, N, K, alpha.data_ptr<float>(), ptr_or_null(ws), ws_bytes, status_ptr(status), stream_of(A)),
        "gemm_ragged");
}

// Walks the vocabulary in pieces of `piece` columns with one [M, piece] buffer: the piece's softmax gradient, then its
// rows of dweight, then its share of dx, summed over the pieces in fp32.  `r` has the forward's x, and its target or, with live,
// the labels put first; the rows are put first again here (that copy is small beside the products, but not beside what the node
// keeps).
OptPair run_ce_backward(const Tensor& dloss, const Tensor& inv_count, const Tensor& lse, const CeRows& r, const Tensor& weight,
                        int64_t ignore_index, int64_t piece, bool need_dx, bool need_dw, const Tensor& status) {
  const Tensor& x = r.x;
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t M = x.size(0), V = weight.size(0), K = x.size(1);
  OptTensor dx, dw, dx32;
  if (M == 0) {
    if (need_dx) dx = at::zeros_like(x);
    if (need_dw) dw = at::zeros_like(weight);
    return {dx, dw};
  }
  const int32_t* live = live_ptr(r.live);
  Tensor xs = x.as_strided({M, K}, {K, 1});
  const Tensor ws = weight.as_strided({V, K}, {K, 1});
  if (live != nullptr) {
    xs = new_matrix(x, M, K, at::kBFloat16);
    check(coda_b200_ce_gather(x.data_ptr(), r.position.data_ptr<int32_t>(), live, xs.data_ptr(), static_cast<int>(M), static_cast<int>(K),
                              stream_of(x)),
          "ce_gather");
  }
  const Tensor dl = dloss.to(at::kFloat);
  const Tensor alpha = at::empty({1}, inv_count.options());
  check(coda_b200_ce_alpha(dl.data_ptr<float>(), inv_count.data_ptr<float>(), alpha.data_ptr<float>(), stream_of(x)), "ce_alpha");
  const int64_t width = std::min(piece, V), ldg = (width + 7) / 8 * 8;
  Tensor g = new_matrix(x, M, ldg, at::kBFloat16);
  if (need_dx) dx = new_matrix(x, M, K, at::kBFloat16);
  if (need_dw) dw = new_matrix(x, V, K, at::kBFloat16);
  Tensor counted = xs;  // the rows of the weight gradient
  if (need_dw && live == nullptr) {
    counted = at::empty_like(xs);
    check(coda_b200_ce_mask(xs.data_ptr(), r.target.data_ptr<int32_t>(), static_cast<int>(ignore_index), counted.data_ptr(),
                            static_cast<int>(M), static_cast<int>(K), stream_of(x)),
          "ce_mask");
  }
  if (need_dx && width < V) dx32 = new_matrix(x, M, K, at::kFloat);
  for (int64_t c0 = 0; c0 < V; c0 += width) {
    const int64_t n = std::min(width, V - c0);
    const Tensor w = ws.narrow(0, c0, n), gp = g.as_strided({M, n}, {ldg, 1});
    check(coda_b200_gemm_softmax_grad(xs.data_ptr(), K, 1, w.data_ptr(), 1, K, lse.data_ptr<float>(), r.target.data_ptr<int32_t>(),
                                      static_cast<int>(ignore_index), static_cast<int>(c0), live, gp.data_ptr(), ldg, static_cast<int>(M),
                                      static_cast<int>(n), static_cast<int>(K), status_ptr(status), stream_of(x)),
          "gemm_softmax_grad");
    if (need_dw) {
      Tensor out = dw->narrow(0, c0, n);
      if (live == nullptr)
        gemm_ragged(gp.t(), counted, out, alpha, c10::nullopt, status);
      else
        check(coda_b200_gemm_live(gp.data_ptr(), ldg, xs.data_ptr(), K, nullptr, out.data_ptr(), K, 0, alpha.data_ptr<float>(), live, 1,
                                  static_cast<int>(n), static_cast<int>(K), static_cast<int>(M), status_ptr(status), stream_of(x)),
              "gemm_live");
    }
    if (need_dx) {
      const bool last = c0 + n == V;
      Tensor out = last ? *dx : *dx32;
      // a product with so few tiles that its last round is cut along the contraction runs over all rows (what it makes of the
      // others is not looked at): 1003 x 1032 x 32003, 404 us a step instead of 613
      const bool cut = c0 == 0 && coda_b200_gemm_workspace_bytes(static_cast<int>(M), static_cast<int>(K), static_cast<int>(n)) > 0;
      if (live == nullptr || cut)
        gemm_ragged(gp, w, out, alpha, c0 > 0 ? dx32 : c10::nullopt, status);
      else
        check(coda_b200_gemm_live(gp.data_ptr(), ldg, w.data_ptr(), K, c0 > 0 ? dx32->data_ptr<float>() : nullptr, out.data_ptr(), K, !last,
                                  alpha.data_ptr<float>(), live, 0, static_cast<int>(M), static_cast<int>(K), static_cast<int>(n),
                                  status_ptr(status), stream_of(x)),
              "gemm_live");
    }
  }
  if (need_dx && live != nullptr) {  // into the memory of the rows, which are not needed any more
    check(coda_b200_ce_scatter(dx->data_ptr(), r.position.data_ptr<int32_t>(), xs.data_ptr(), static_cast<int>(M), static_cast<int>(K),
                               stream_of(x)),
          "ce_scatter");
    dx = xs;
  }
  return {dx, dw};
}

inline void require_ce(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t ignore_index) {
  for (const Tensor* t : {&x, &weight}) {
    require_cuda(*t);
    TORCH_CHECK_NOT_IMPLEMENTED(t->scalar_type() == at::kBFloat16, "coda_b200 operators take bfloat16 matrices, got ", t->scalar_type());
  }
  TORCH_CHECK_VALUE(x.dim() == 2 && weight.dim() == 2 && x.size(1) == weight.size(1), "x [M, K] and weight [V, K] expected");
  TORCH_CHECK_VALUE(weight.size(0) > 0 && x.size(1) > 0 && x.size(1) % 8 == 0, "weight must have rows, and K must be a positive multiple of 8");
  TORCH_CHECK_VALUE(target.device() == x.device() && weight.device() == x.device(), "x, weight and target must be on one device");
  TORCH_CHECK_VALUE(target.dim() == 1 && target.size(0) == x.size(0) && target.scalar_type() == at::kInt, "target must have one label per row");
  TORCH_CHECK_VALUE(ignore_index >= INT_MIN && ignore_index <= INT_MAX, "ignore_index must fit int32");
  TORCH_CHECK_VALUE(x.size(0) <= INT_MAX && weight.size(0) <= INT_MAX - 256, "extents must fit 31 bits");
}

// (loss, inv_count, lse, and with `compact` the counted rows' labels, put first as lse is, position and live).  Whether to is
// the caller's to say: a recorded program keeps what it was recorded with, whatever the options are when it runs.
std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor, OptTensor> ce_pieces_fwd(const Tensor& x, const Tensor& weight, const Tensor& target,
                                                                                 int64_t ignore_index, bool mean, bool compact,
                                                                                 const Tensor& status) {
  require_ce(x, weight, target, ignore_index);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(x.device());
  const CeRows r = ce_rows(aligned16(x), target.contiguous(), ignore_index, compact && x.size(0) > 0);
  auto [loss, inv_count, lse] = run_ce(r, aligned16(weight), ignore_index, mean, status);
  if (!r.live.defined()) return {loss, inv_count, lse, c10::nullopt, c10::nullopt, c10::nullopt};
  return {loss, inv_count, lse, r.target, r.position, r.live};
}

// x: the forward's; target too, or the labels it put first, with position and live
OptPair ce_pieces_bwd(const Tensor& dloss, const Tensor& inv_count, const Tensor& lse, const Tensor& x, const Tensor& weight,
                      const Tensor& target, const OptTensor& position, const OptTensor& live, int64_t ignore_index, int64_t piece, bool need_dx,
                      bool need_dw, const Tensor& status) {
  require_ce(x, weight, target, ignore_index);
  TORCH_CHECK_VALUE(piece >= 1, "piece must be at least 1");
  for (const Tensor* t : {&inv_count, &lse})
    TORCH_CHECK_VALUE(t->device() == x.device() && t->scalar_type() == at::kFloat && t->is_contiguous(), "float32 statistics expected");
  TORCH_CHECK_VALUE(inv_count.numel() == 1 && dloss.numel() == 1 && lse.numel() == x.size(0), "one dloss, inv_count, and one lse a row expected");
  TORCH_CHECK_VALUE(position.has_value() == live.has_value(), "position and live belong together");
  if (live.has_value())
    TORCH_CHECK_VALUE(position->device() == x.device() && position->scalar_type() == at::kInt && position->is_contiguous() &&
                          position->numel() == x.size(0) && live->device() == x.device() && live->scalar_type() == at::kInt && live->numel() == 1,
                      "position must be int32 with one entry per row, live one int32");
  at::AutoDispatchBelowADInplaceOrView below;
  return run_ce_backward(dloss, inv_count, lse, CeRows{aligned16(x), target.contiguous(), position.value_or(Tensor()), live.value_or(Tensor())},
                         aligned16(weight), ignore_index, piece, need_dx, need_dw, status);
}

Tensor linear_cross_entropy_pieces(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t ignore_index, bool mean, int64_t,
                                   const Tensor& status) {
  return std::get<0>(ce_pieces_fwd(x, weight, target, ignore_index, mean, ce_compacts(x, weight), status));
}

// ---------------------------------------------------------------------------------------- their gradients
namespace autograd {

Tensor call_dropout(const Tensor& x, double p, const OptTensor& rng, int64_t stream) {
  static const auto op = operator_named<Tensor(const Tensor&, double, const OptTensor&, int64_t)>("coda_b200n::dropout");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, p, rng, stream);
}
auto call_norm_fwd(const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps, double p, const OptTensor& rng, int64_t stream,
                   bool keep_low) {
  static const auto op = operator_named<std::tuple<Tensor, OptTensor, Tensor, OptTensor, OptTensor>(
      const Tensor&, const OptTensor&, const Tensor&, double, double, const OptTensor&, int64_t, bool)>("coda_b200n::norm_fwd");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, residual, weight, eps, p, rng, stream, keep_low);
}
auto call_norm_bwd(const OptTensor& dout, const OptTensor& dh, const Tensor& h, const OptTensor& low, const Tensor& rstd, const Tensor& weight,
                   double p, const OptTensor& rng, int64_t stream, bool need_dx, bool need_dres, bool need_dw) {
  static const auto op = operator_named<std::tuple<OptTensor, OptTensor, OptTensor>(
      const OptTensor&, const OptTensor&, const Tensor&, const OptTensor&, const Tensor&, const Tensor&, double, const OptTensor&, int64_t, bool,
      bool, bool)>("coda_b200n::norm_bwd");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(dout, dh, h, low, rstd, weight, p, rng, stream, need_dx, need_dres, need_dw);
}

class DropoutNode : public torch::autograd::Function<DropoutNode> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, const OptTensor& rng, int64_t stream) {
    static const auto op =
        operator_named<std::tuple<Tensor, Tensor>(const Tensor&, double, const OptTensor&, int64_t)>("coda_b200n::dropout_fwd");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, used] = op.call(x, p, rng, stream);
    ctx->save_for_backward({used});
    ctx->saved_data["p"] = p;
    ctx->saved_data["stream"] = stream;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    require_first_order("dropout");
    const Tensor used = ctx->get_saved_variables()[0];
    return {call_dropout(grads[0], ctx->saved_data["p"].toDouble(), used, ctx->saved_data["stream"].toInt()), Tensor(), Tensor(), Tensor()};
  }
};

class RMSNormNode : public torch::autograd::Function<RMSNormNode> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& weight, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x = x_in.contiguous();
    auto f = call_norm_fwd(x, c10::nullopt, weight, eps, 0.0, c10::nullopt, 0, false);
    ctx->save_for_backward({x, weight, std::get<2>(f)});
    return std::get<0>(f);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    require_first_order("rms_norm");
    const auto saved = ctx->get_saved_variables();
    auto g = call_norm_bwd(grads[0], c10::nullopt, saved[0], c10::nullopt, saved[2], saved[1], 0.0, c10::nullopt, 0, false,
                           ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    return {std::get<1>(g).value_or(Tensor()), std::get<2>(g).value_or(Tensor()), Tensor()};
  }
};

class AddRMSNormNode : public torch::autograd::Function<AddRMSNormNode> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& weight, double eps, double p,
                               const OptTensor& rng, int64_t stream) {
    auto f = call_norm_fwd(x, residual, weight, eps, p, rng, stream, true);
    const Tensor &out = std::get<0>(f), &h = *std::get<1>(f);
    ctx->save_for_backward({h, weight, std::get<2>(f), std::get<3>(f).value_or(Tensor()), std::get<4>(f).value_or(Tensor())});
    ctx->saved_data["p"] = p;
    ctx->saved_data["stream"] = stream;
    ctx->set_materialize_grads(false);
    return {out, h};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    require_first_order("add_rms_norm");
    const auto saved = ctx->get_saved_variables();
    auto g = call_norm_bwd(optional(grads[0]), optional(grads[1]), saved[0], optional(saved[4]), saved[2], saved[1],
                           ctx->saved_data["p"].toDouble(), optional(saved[3]), ctx->saved_data["stream"].toInt(), ctx->needs_input_grad(0),
                           ctx->needs_input_grad(1), ctx->needs_input_grad(2));
    return {std::get<0>(g).value_or(Tensor()), std::get<1>(g).value_or(Tensor()), std::get<2>(g).value_or(Tensor()), Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};

class CePiecesNode : public torch::autograd::Function<CePiecesNode> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& weight_in, const Tensor& target_in, int64_t ignore_index,
                        bool mean, int64_t piece, const Tensor& status) {
    static const auto op = operator_named<std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor, OptTensor>(
        const Tensor&, const Tensor&, const Tensor&, int64_t, bool, bool, const Tensor&)>("coda_b200n::ce_pieces_fwd");
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x = x_in.contiguous(), weight = weight_in.contiguous(), target = target_in.contiguous();
    auto [loss, inv_count, lse, labels, position, live] = op.call(x, weight, target, ignore_index, mean, ce_compacts(x, weight), status);
    ctx->save_for_backward({x, weight, labels.value_or(target), lse, inv_count, position.value_or(Tensor()), live.value_or(Tensor())});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["piece"] = piece;
    ctx->saved_data["status"] = status;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto op = operator_named<OptPair(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                  const OptTensor&, const OptTensor&, int64_t, int64_t, bool, bool, const Tensor&)>(
        "coda_b200n::ce_pieces_bwd");
    require_first_order("linear_cross_entropy_pieces");
    const auto s = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dx, dw] = op.call(grads[0], s[4], s[3], s[0], s[1], s[2], optional(s[5]), optional(s[6]), ctx->saved_data["ignore_index"].toInt(),
                            ctx->saved_data["piece"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                            ctx->saved_data["status"].toTensor());
    return {dx.value_or(Tensor()), dw.value_or(Tensor()), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor dropout(const Tensor& x, double p, const OptTensor& rng, int64_t stream) {
  require_no_tangent("dropout", {&x});
  return wants_grad({&x}) ? DropoutNode::apply(x, p, rng, stream) : call_dropout(x, p, rng, stream);
}

Tensor rms_norm(const Tensor& x, const Tensor& weight, double eps) {
  static const auto op = operator_named<Tensor(const Tensor&, const Tensor&, double)>("coda_b200n::rms_norm");
  require_no_tangent("rms_norm", {&x, &weight});
  if (wants_grad({&x, &weight})) return RMSNormNode::apply(x, weight, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, eps);
}

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps, double p,
                                        const OptTensor& rng, int64_t stream) {
  static const auto op = operator_named<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, double, double, const OptTensor&,
                                                                   int64_t)>("coda_b200n::add_rms_norm");
  require_no_tangent("add_rms_norm", {&x, &residual, &weight});
  if (wants_grad({&x, &residual, &weight})) {
    auto r = AddRMSNormNode::apply(x, residual, weight, eps, p, rng, stream);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, residual, weight, eps, p, rng, stream);
}

std::tuple<Tensor, Tensor, OptTensor> rows_e4m3(const Tensor& x, const OptTensor& residual, const OptTensor& weight, double eps) {
  static const auto op = operator_named<std::tuple<Tensor, Tensor, OptTensor>(const Tensor&, const OptTensor&, const OptTensor&, double)>(
      "coda_b200n::rows_e4m3");
  const Tensor none;
  require_no_grad("the e4m3 output", {&x, residual.has_value() ? &*residual : &none, weight.has_value() ? &*weight : &none});
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, residual, weight, eps);
}

Tensor linear_e4m3(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& weight_scale, bool out_fp32, const Tensor& status) {
  static const auto op =
      operator_named<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, bool, const Tensor&)>("coda_b200n::linear_e4m3");
  require_no_grad("linear_e4m3", {&x, &x_scale, &weight, &weight_scale});
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, x_scale, weight, weight_scale, out_fp32, status);
}

Tensor linear_cross_entropy_pieces(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t ignore_index, bool mean, int64_t piece,
                                   const Tensor& status) {
  static const auto op = operator_named<Tensor(const Tensor&, const Tensor&, const Tensor&, int64_t, bool, int64_t, const Tensor&)>(
      "coda_b200n::linear_cross_entropy_pieces");
  require_no_tangent("linear_cross_entropy_pieces", {&x, &weight});
  if (wants_grad({&x, &weight})) return CePiecesNode::apply(x, weight, target, ignore_index, mean, piece, status);
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, target, ignore_index, mean, piece, status);
}

}  // namespace autograd
}  // namespace

TORCH_LIBRARY(coda_b200n, m) {
  m.def("gemm_out(Tensor A, Tensor B, Tensor(a!) out, Tensor? alpha, Tensor? C, Tensor status) -> ()");
  m.def("gemm_sigmoid_out(Tensor A, Tensor B, Tensor(a!) out, Tensor status) -> ()");
  m.def("gemm_swiglu_out(Tensor A, Tensor B, Tensor(a!) preact, Tensor(b!) postact, Tensor status) -> ()");
  m.def("gemm_lse_out(Tensor A, Tensor B, Tensor(a!)? probs, Tensor(b!) part_max, Tensor(c!) part_sum, Tensor target, "
        "Tensor(d!) target_logit, Tensor status) -> ()");
  m.def("lse_finalize_out(Tensor part_max, Tensor part_sum, Tensor target, Tensor target_logit, int ignore_index, "
        "Tensor(a!) lse, Tensor(b!) losses) -> ()");
  m.def("ce_grad_fixup_(Tensor(a!) probs, Tensor part_max, Tensor lse, Tensor target, int ignore_index) -> ()");
  m.def("gemm_qknorm_rope_out(Tensor A, Tensor B, Tensor(a!) qk, Tensor(b!) preact, Tensor(c!)? v, Tensor(d!) mean_sq, Tensor gamma, "
        "Tensor positions, Tensor frequencies, int head_dim, int num_heads_q, int num_heads_k, float eps, Tensor status) -> ()");
  m.def("dswiglu_out(Tensor preact, Tensor dout, Tensor(a!) grad_pre) -> ()");
  m.def("dsigmoid_out(Tensor out, Tensor dout, Tensor(a!) grad_pre) -> ()");
  m.def("qknorm_rope_bwd_out(Tensor dq, Tensor dk, Tensor? dv, Tensor preact, Tensor mean_sq, Tensor gamma, Tensor positions, "
        "Tensor frequencies, int head_dim, int num_heads_q, int num_heads_k, float eps, Tensor(a!) grad, Tensor(b!) dgamma, "
        "Tensor(c!) scratch) -> ()");

  m.def("linear_backward(Tensor grad_pre, Tensor x, Tensor weight, bool need_dx, bool need_dw, Tensor? alpha, Tensor status) -> "
        "(Tensor?, Tensor?)");
  m.def("swiglu_fwd(Tensor x, Tensor weight, Tensor status) -> (Tensor, Tensor)");
  m.def("swiglu_bwd(Tensor preact, Tensor dout, Tensor x, Tensor weight, bool need_dx, bool need_dw, Tensor status) -> (Tensor?, Tensor?)");
  m.def("sigmoid_fwd(Tensor x, Tensor weight, bool out_fp32, Tensor status) -> Tensor");
  m.def("sigmoid_bwd(Tensor out, Tensor dout, Tensor x, Tensor weight, bool need_dx, bool need_dw, Tensor status) -> (Tensor?, Tensor?)");
  m.def("cross_entropy_fwd(Tensor x, Tensor weight, Tensor target, int ignore_index, bool mean, bool store_grad, Tensor status) -> "
        "(Tensor, Tensor?, Tensor?)");
  m.def("cross_entropy_bwd(Tensor dloss, Tensor? inv_count, Tensor dlogits, Tensor x, Tensor weight, bool need_dx, bool need_dw, "
        "Tensor status) -> (Tensor?, Tensor?)");
  m.def("qknorm_rope_fwd(Tensor x, Tensor weight, Tensor gamma, Tensor positions, Tensor frequencies, int head_dim, int num_heads_q, "
        "int num_heads_k, float eps, Tensor status) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("qknorm_rope_bwd(Tensor dq, Tensor dk, Tensor dv, Tensor x, Tensor weight, Tensor preact, Tensor mean_sq, Tensor gamma, "
        "Tensor positions, Tensor frequencies, int head_dim, int num_heads_q, int num_heads_k, float eps, bool need_dx, bool need_dw, "
        "Tensor status) -> (Tensor?, Tensor?, Tensor)");

  m.def("dropout(Tensor x, float p, Tensor? rng, int stream) -> Tensor");
  m.def("dropout_fwd(Tensor x, float p, Tensor? rng, int stream) -> (Tensor, Tensor)");
  m.def("norm_fwd(Tensor x, Tensor? residual, Tensor weight, float eps, float p, Tensor? rng, int stream, bool keep_low) -> "
        "(Tensor, Tensor?, Tensor, Tensor?, Tensor?)");
  m.def("norm_bwd(Tensor? dout, Tensor? dh, Tensor h, Tensor? low, Tensor rstd, Tensor weight, float p, Tensor? rng, int stream, bool need_dx, "
        "bool need_dres, bool need_dw) -> (Tensor?, Tensor?, Tensor?)");
  m.def("ce_pieces_fwd(Tensor x, Tensor weight, Tensor target, int ignore_index, bool mean, bool compact, Tensor status) -> "
        "(Tensor, Tensor, Tensor, Tensor?, Tensor?, Tensor?)");
  m.def("ce_pieces_bwd(Tensor dloss, Tensor inv_count, Tensor lse, Tensor x, Tensor weight, Tensor target, Tensor? position, Tensor? live, "
        "int ignore_index, int piece, bool need_dx, bool need_dw, Tensor status) -> (Tensor?, Tensor?)");
  m.def("rms_norm(Tensor x, Tensor weight, float eps) -> Tensor");
  m.def("add_rms_norm(Tensor x, Tensor residual, Tensor weight, float eps, float p, Tensor? rng, int stream) -> (Tensor, Tensor)");
  m.def("rows_e4m3(Tensor x, Tensor? residual, Tensor? weight, float eps) -> (Tensor, Tensor, Tensor?)");
  m.def("linear_e4m3(Tensor x, Tensor x_scale, Tensor weight, Tensor weight_scale, bool out_fp32, Tensor status) -> Tensor");
  m.def("linear_cross_entropy_pieces(Tensor x, Tensor weight, Tensor target, int ignore_index, bool mean, int piece, Tensor status) -> Tensor");
}

TORCH_LIBRARY_IMPL(coda_b200n, CUDA, m) {
  m.impl("gemm_out", gemm_out);
  m.impl("gemm_sigmoid_out", gemm_sigmoid_out);
  m.impl("gemm_swiglu_out", gemm_swiglu_out);
  m.impl("gemm_lse_out", gemm_lse_out);
  m.impl("lse_finalize_out", lse_finalize_out);
  m.impl("ce_grad_fixup_", ce_grad_fixup_);
  m.impl("gemm_qknorm_rope_out", gemm_qknorm_rope_out);
  m.impl("dswiglu_out", dswiglu_out);
  m.impl("dsigmoid_out", dsigmoid_out);
  m.impl("qknorm_rope_bwd_out", qknorm_rope_bwd_out);
  m.impl("linear_backward", linear_backward);
  m.impl("swiglu_fwd", swiglu_fwd);
  m.impl("swiglu_bwd", swiglu_bwd);
  m.impl("sigmoid_fwd", sigmoid_fwd);
  m.impl("sigmoid_bwd", sigmoid_bwd);
  m.impl("cross_entropy_fwd", cross_entropy_fwd);
  m.impl("cross_entropy_bwd", cross_entropy_bwd);
  m.impl("qknorm_rope_fwd", qknorm_rope_fwd);
  m.impl("qknorm_rope_bwd", qknorm_rope_bwd);
}

TORCH_LIBRARY_IMPL(coda_b200n, CUDA, m) {
  m.impl("dropout", dropout);
  m.impl("dropout_fwd", dropout_fwd);
  m.impl("norm_fwd", norm_fwd);
  m.impl("norm_bwd", norm_bwd);
  m.impl("rms_norm", rms_norm);
  m.impl("add_rms_norm", add_rms_norm);
  m.impl("rows_e4m3", rows_e4m3);
  m.impl("linear_e4m3", linear_e4m3);
  m.impl("ce_pieces_fwd", ce_pieces_fwd);
  m.impl("ce_pieces_bwd", ce_pieces_bwd);
  m.impl("linear_cross_entropy_pieces", linear_cross_entropy_pieces);
}
TORCH_LIBRARY_IMPL(coda_b200n, AutogradCUDA, m) {
  m.impl("dropout", autograd::dropout);
  m.impl("rms_norm", autograd::rms_norm);
  m.impl("add_rms_norm", autograd::add_rms_norm);
  m.impl("rows_e4m3", autograd::rows_e4m3);
  m.impl("linear_e4m3", autograd::linear_e4m3);
  m.impl("linear_cross_entropy_pieces", autograd::linear_cross_entropy_pieces);
}
