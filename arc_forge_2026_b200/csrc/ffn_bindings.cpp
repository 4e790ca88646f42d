// Bindings of the gated feed-forward block, the norms with trainable weights and dropout: argument checks,
// allocation of results and scratch on the tensors' own device, launch on that device's current stream, and their
// autograd nodes (in C++: a small call's time is the host's, and a Python node costs several times the kernels).
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "binding_utils.h"
#include "ffn.h"

using namespace afb_bind;

namespace {

using OptT = c10::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptT& t) { return t.has_value() && wants_grad(*t); }
at::Tensor val(const OptT& t) { return t.has_value() ? *t : at::Tensor(); }
OptT opt(const at::Tensor& t) { return t.defined() ? OptT(t) : OptT(); }
// Whether a tensor's memory holds its value. It does not where the tensor is a function transform's wrapper, dispatches
// to Python (a fake tensor has no memory at all), or is negated, conjugated or zeroed only when it is read.
bool in_memory(const at::Tensor& t) {
  using K = c10::DispatchKey;
  static const c10::DispatchKeySet lazy({K::Python, K::Negative, K::Conjugate, K::ZeroTensor, K::Functionalize,
                                         K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Batched});
  return !t.key_set().has_any(lazy);
}
bool in_memory(const OptT& t) { return !t.has_value() || in_memory(*t); }
// a tensor that carries a tangent (forward-mode differentiation; it need not require a gradient)
bool dual(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }
bool dual(const OptT& t) { return t.has_value() && dual(*t); }
// Whether operations have to go through the dispatcher: inside a function transform, under a dispatch mode or while a
// trace is recorded, where a kernel launch would pass unseen. There and for dual tensors, whose tangents the kernels do not
// make, the callers take their plain forms, and backward passes the formulas in ordinary operations.
bool dispatched() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing() ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}
template <class... Ts>
bool launchable(const Ts&... ts) {
  return (in_memory(ts) && ...) && !(dual(ts) || ...) && !dispatched();
}
// x with its leading dimensions as one
at::Tensor rows2d(const at::Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }
void differentiable_once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once: create_graph=True is not supported");
}

// A leaf's gradient goes to its accumulator on the stream on which the leaf was first used by a graph that still lives.
// Where that is the default stream, a capture on another one would have to be joined by it, which CUDA forbids (and the
// error can end the process): refused here, before it comes to that.
void capturable_backward(const char* what) {
  const auto node = torch::autograd::get_current_node();
  const auto st = at::cuda::getCurrentCUDAStream();
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (!node || st.stream() == nullptr || cudaStreamIsCapturing(st.stream(), &status) != cudaSuccess ||
      status == cudaStreamCaptureStatusNone)
    return;
  for (const auto& e : node->next_edges())
    if (auto* acc = dynamic_cast<torch::autograd::AccumulateGrad*>(e.function.get())) {
      const auto s = acc->stream();
      TORCH_CHECK(!s || s->id() != 0, what, ": its backward pass is captured while a graph of the same leaf that was made",
                  " outside the capture, on the default stream, is alive; release that graph first");
    }
}

int elem_type(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return afb::ELEM_BF16;
    case at::kHalf: return afb::ELEM_FP16;
    case at::kFloat: return afb::ELEM_FP32;
    default: TORCH_CHECK(false, what, ": bf16, fp16 or fp32 expected, got ", t.scalar_type());
  }
}

// rows a TMA tensor map can walk: unit inner stride, row stride a multiple of 16 bytes, 16-byte aligned base; copied
// into that form when they are not
at::Tensor tma_rows(const at::Tensor& t) {
  const int64_t e = t.element_size();
  const bool ok = t.stride(1) == 1 && (t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) * e % 16 == 0)) &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (ok) return t;
  at::Tensor c = at::empty(t.sizes(), t.options());
  c.copy_(t);
  return c;
}
int64_t ld(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

afb::FfnShape ffn_shape(const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w2, int64_t act) {
  AFB_CHECK_CUDA(x);
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "gated_ffn: bf16 or fp16 x");
  TORCH_CHECK(x.dim() == 2 && w13.dim() == 2 && w2.dim() == 2, "gated_ffn: x [T, H], w13 [2F, H], w2 [N, F]");
  TORCH_CHECK(w13.size(1) == x.size(1) && w13.size(0) == 2 * w2.size(1), "gated_ffn: x [T, H], w13 [2F, H], w2 [N, F]");
  TORCH_CHECK(x.size(1) > 0 && w2.size(1) > 0 && w2.size(0) > 0 && x.size(1) % 8 == 0 && w2.size(1) % 8 == 0 &&
                  w2.size(0) % 8 == 0,
              "gated_ffn: H, F and N are multiples of 8");
  TORCH_CHECK(x.size(0) < (int64_t(1) << 31) - 1024 && x.size(1) < (1 << 22) && w13.size(0) < (1 << 22) &&
                  w2.size(0) < (1 << 22),
              "gated_ffn: size out of range");
  TORCH_CHECK(act >= 0 && act <= 2, "gated_ffn: act is 0 (silu), 1 (tanh-GELU) or 2 (erf-GELU)");
  for (const at::Tensor* t : {&w13, &w2})
    TORCH_CHECK(t->device() == x.device() && t->scalar_type() == x.scalar_type(),
                "gated_ffn: weights are on x's device, in its type");
  afb::FfnShape s;
  s.T = x.size(0), s.H = (int)x.size(1), s.F = (int)w2.size(1), s.N = (int)w2.size(0);
  s.act = (int)act, s.fp16 = x.scalar_type() == at::kHalf;
  return s;
}

at::Tensor scratch_of(size_t n, const at::Tensor& like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kFloat));
}

// (y, h, gu): h and gu are what ffn_bwd reads; gu is kept only when `save`. y has x's leading dimensions (made in that
// shape: a view as the result of an autograd node could not be changed in place).
std::tuple<at::Tensor, at::Tensor, OptT> gated_ffn_fwd(const at::Tensor& xn, const at::Tensor& w13_,
                                                       const at::Tensor& w2_, const OptT& rn, int64_t act, bool save) {
  const at::Tensor x_ = rows2d(xn);
  const OptT residual = rn ? OptT(rows2d(*rn)) : OptT();
  const afb::FfnShape s = ffn_shape(x_, w13_, w2_, act);
  c10::cuda::CUDAGuard g(x_.device());
  const at::Tensor x = tma_rows(x_), w13 = tma_rows(w13_.contiguous()), w2 = tma_rows(w2_.contiguous());
  at::Tensor r;
  if (residual.has_value()) {
    TORCH_CHECK(residual->dim() == 2 && residual->size(0) == s.T && residual->size(1) == s.N &&
                    residual->scalar_type() == x.scalar_type() && residual->device() == x.device(),
                "gated_ffn: residual is [T, N] in x's type on its device");
    r = tma_rows(*residual);
  }
  auto shape = xn.sizes().vec();
  shape.back() = s.N;
  at::Tensor y = at::empty(shape, x.options()), h = at::empty({afb::ffn_h_rows(s), s.F}, x.options());
  OptT gu;
  if (save) gu = at::empty({(s.T + 31) / 32 * 32, 2 * (int64_t)s.F}, x.options().dtype(at::kFloat));
  const size_t n_scr = afb::ffn_fwd_scratch(s, num_sms());
  const at::Tensor scr = n_scr ? scratch_of(n_scr, x) : at::Tensor();
  check_rc(afb::ffn_fwd(s, x.data_ptr(), ld(x), w13.data_ptr(), w2.data_ptr(), r.defined() ? r.data_ptr() : nullptr,
                        r.defined() ? ld(r) : 0, h.data_ptr(), optr<float>(gu), y.data_ptr(),
                        n_scr ? ptr<float>(scr) : nullptr, num_sms(), status_ptr(x.get_device()), stream()),
           "gated_ffn_fwd");
  return {y, h, gu};
}

// (dx, dw13, dw2), each None unless asked for
std::tuple<OptT, OptT, OptT> gated_ffn_bwd(const at::Tensor& dy_, const at::Tensor& x_, const at::Tensor& w13_,
                                           const at::Tensor& w2_, OptT h, OptT gu, int64_t act, bool need_dx,
                                           bool need_dw13, bool need_dw2) {
  const afb::FfnShape s = ffn_shape(x_, w13_, w2_, act);
  TORCH_CHECK(dy_.dim() == 2 && dy_.size(0) == s.T && dy_.size(1) == s.N && dy_.scalar_type() == x_.scalar_type() &&
                  dy_.device() == x_.device(),
              "gated_ffn: dy is [T, N] in x's type on its device");
  if (need_dw2)
    TORCH_CHECK(h.has_value() && h->is_contiguous() && h->scalar_type() == x_.scalar_type() && h->dim() == 2 &&
                    h->size(0) >= s.T && h->size(1) == s.F && h->device() == x_.device(),
                "gated_ffn: h of the forward pass");
  if (need_dx || need_dw13)
    TORCH_CHECK(gu.has_value() && gu->is_contiguous() && gu->scalar_type() == at::kFloat && gu->dim() == 2 &&
                    gu->size(0) >= s.T && gu->size(1) == 2 * (int64_t)s.F && gu->device() == x_.device(),
                "gated_ffn: gu of the forward pass");
  c10::cuda::CUDAGuard g(x_.device());
  const at::Tensor x = tma_rows(x_), w13 = tma_rows(w13_.contiguous()), w2 = tma_rows(w2_.contiguous()),
                   dy = tma_rows(dy_);
  OptT dx, dw13, dw2;
  at::Tensor dgu;
  if (need_dx || need_dw13) dgu = at::empty({s.T, 2 * (int64_t)s.F}, x.options());
  if (need_dx) dx = at::empty({s.T, s.H}, x.options());
  if (need_dw13) dw13 = at::empty({2 * (int64_t)s.F, s.H}, x.options());
  if (need_dw2) dw2 = at::empty({s.N, s.F}, x.options());
  if (s.T == 0) {
    if (dw13) dw13->zero_();
    if (dw2) dw2->zero_();
    return {dx, dw13, dw2};
  }
  const at::Tensor scr = scratch_of(afb::ffn_bwd_scratch(s, num_sms()), x);
  check_rc(afb::ffn_bwd(s, dy.data_ptr(), ld(dy), x.data_ptr(), ld(x), w13.data_ptr(), w2.data_ptr(), optr<void>(h),
                        optr<float>(gu), dgu.defined() ? dgu.data_ptr() : nullptr, optr<void>(dx), optr<void>(dw13),
                        optr<void>(dw2), ptr<float>(scr), num_sms(), status_ptr(x.get_device()), stream()),
           "gated_ffn_bwd");
  return {dx, dw13, dw2};
}

afb::NormArgs norm_args(const at::Tensor& x, const at::Tensor& w, bool rms, double eps) {
  AFB_CHECK_CUDA(x);
  TORCH_CHECK(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) == 1), "norm: x is [rows, width] with unit inner stride");
  afb::NormArgs a;
  a.rows = x.size(0), a.width = (int)x.size(1), a.rms = rms, a.eps = (float)eps;
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= afb::NORM_MAX_WIDTH, "norm: rows of 1 to ", afb::NORM_MAX_WIDTH);
  a.dtype = elem_type(x, "norm x");
  a.wtype = elem_type(w, "norm w");
  TORCH_CHECK(a.wtype == a.dtype || a.wtype == afb::ELEM_FP32, "norm: weights in x's type or fp32");
  TORCH_CHECK(w.device() == x.device() && w.dim() == 1 && w.size(0) == x.size(1) && w.is_contiguous(),
              "norm: w is contiguous [width] on x's device");
  a.x = x.data_ptr(), a.ldx = x.stride(0), a.w = w.data_ptr();
  a.status = status_ptr(x.get_device());
  return a;
}

// x [..., width] as rows with unit inner stride
at::Tensor norm_rows(const at::Tensor& x) {
  const at::Tensor r = rows2d(x);
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

// (y, mean, rstd); mean and rstd only when `save` (mean not for rms); y has x's shape
std::tuple<at::Tensor, OptT, OptT> norm_train_fwd(const at::Tensor& xn, const at::Tensor& w, OptT b, double eps,
                                                  bool rms, bool save) {
  const at::Tensor x = norm_rows(xn);
  afb::NormArgs a = norm_args(x, w, rms, eps);
  if (b.has_value()) {
    TORCH_CHECK(!rms, "norm: rms has no bias");
    TORCH_CHECK(b->device() == x.device() && b->sizes() == w.sizes() && b->scalar_type() == w.scalar_type() &&
                    b->is_contiguous(),
                "norm: b is like w");
    a.b = b->data_ptr();
  }
  c10::cuda::CUDAGuard g(x.device());
  at::Tensor y = at::empty(xn.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  OptT mean, rstd;
  if (save) {
    rstd = at::empty({a.rows}, x.options().dtype(at::kFloat));
    if (!rms) mean = at::empty({a.rows}, x.options().dtype(at::kFloat));
  }
  a.y = y.data_ptr(), a.mean = optr<float>(mean), a.rstd = optr<float>(rstd);
  check_rc(afb::norm_fwd(a, num_sms(), stream()), "norm_train_fwd");
  return {y, mean, rstd};
}

// (dx, dw, db), each None unless asked for
std::tuple<OptT, OptT, OptT> norm_train_bwd(const at::Tensor& dy_, const at::Tensor& x, const at::Tensor& w, OptT mean,
                                            const at::Tensor& rstd, bool rms, bool need_dx, bool need_dw,
                                            bool need_db) {
  afb::NormArgs a = norm_args(x, w, rms, 0.);
  TORCH_CHECK(dy_.sizes() == x.sizes() && dy_.scalar_type() == x.scalar_type() && dy_.device() == x.device(),
              "norm: dy is like x");
  TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == a.rows &&
                  rstd.device() == x.device(),
              "norm: rstd of the forward pass");
  TORCH_CHECK(rms || (mean.has_value() && mean->scalar_type() == at::kFloat && mean->is_contiguous() &&
                      mean->numel() == a.rows && mean->device() == x.device()),
              "norm: mean of the forward pass");
  c10::cuda::CUDAGuard g(x.device());
  const at::Tensor dy = dy_.contiguous();
  OptT dx, dw, db;
  if (need_dx) dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  if (need_dw) dw = at::empty(w.sizes(), w.options());
  if (need_db) db = at::empty(w.sizes(), w.options());
  if (a.rows == 0) {
    if (dw) dw->zero_();
    if (db) db->zero_();
    return {dx, dw, db};
  }
  a.dy = dy.data_ptr(), a.mean = optr<float>(mean), a.rstd = ptr<float>(rstd);
  a.dx = optr<void>(dx), a.dw = optr<void>(dw), a.db = optr<void>(db);
  at::Tensor part;
  if (need_dw || need_db) {
    a.partials = afb::norm_bwd_partials(a, num_sms());
    TORCH_CHECK(a.partials > 0, "norm_train_bwd: no launch plan");
    part = scratch_of((size_t)a.partials * 2 * a.width, x);
    a.partial = ptr<float>(part);
  }
  check_rc(afb::norm_bwd(a, num_sms(), stream()), "norm_train_bwd");
  return {dx, dw, db};
}

at::Tensor dropout_op(const at::Tensor& x_, OptT residual, int64_t threshold, int64_t seed, int64_t offset, OptT rng) {
  AFB_CHECK_CUDA(x_);
  const int dt = elem_type(x_, "dropout x");
  TORCH_CHECK(threshold >= 0 && threshold <= 65536, "dropout: threshold out of range");
  c10::cuda::CUDAGuard g(x_.device());
  const at::Tensor x = x_.contiguous();
  at::Tensor r;
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() &&
                    residual->device() == x.device(),
                "dropout: residual is like x");
    r = residual->contiguous();
  }
  const int64_t* rp = nullptr;
  if (rng.has_value()) {
    TORCH_CHECK(rng->scalar_type() == at::kLong && rng->dim() == 1 && rng->numel() == 2 && rng->is_contiguous() &&
                    rng->device() == x.device(),
                "dropout: the seed tensor is int64 [2] (seed, offset) on x's device");
    rp = rng->data_ptr<int64_t>();
  }
  at::Tensor y = at::empty(x.sizes(), x.options());
  check_rc(afb::dropout(x.data_ptr(), r.defined() ? r.data_ptr() : nullptr, y.data_ptr(), x.numel(), dt,
                        (uint32_t)threshold, (uint64_t)seed, (uint64_t)offset, rp, num_sms(), stream()),
           "dropout");
  return y;
}

// ------------------------------------------------------------------------------------------ autograd
struct GatedFfn : torch::autograd::Function<GatedFfn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w2,
                            const OptT& residual, int64_t act) {
    const bool need_gu = wants_grad(x) || wants_grad(w13);
    auto [y, h, gu] = gated_ffn_fwd(x, w13, w2, residual, act, need_gu);
    ctx->save_for_backward({x, w13, w2, wants_grad(w2) ? h : at::Tensor(), val(gu)});
    ctx->saved_data["act"] = act;
    ctx->saved_data["residual"] = residual.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    differentiable_once("gated_ffn");
    capturable_backward("gated_ffn");
    const variable_list v = ctx->get_saved_variables();
    const at::Tensor& dy = grads[0];
    const bool need_x = ctx->needs_input_grad(0), need_w13 = ctx->needs_input_grad(1),
               need_w2 = ctx->needs_input_grad(2);
    variable_list out(5);
    if (!launchable(dy)) {
      const int64_t act = ctx->saved_data["act"].toInt(), F = v[2].size(1);
      const at::Tensor x = v[0].to(at::kFloat), w13 = v[1].to(at::kFloat), w2 = v[2].to(at::kFloat), d = dy.to(at::kFloat);
      const at::Tensor gu = at::matmul(x, w13.t()), g = gu.narrow(-1, 0, F), u = gu.narrow(-1, F, F), one = at::ones_like(g);
      const char* kind = act == 1 ? "tanh" : "none";
      const at::Tensor a = act == 0 ? at::silu(g) : at::gelu(g, kind);
      const at::Tensor da = act == 0 ? at::silu_backward(one, g) : at::gelu_backward(one, g, kind);
      const at::Tensor dh = at::matmul(d, w2), dgu = at::cat({dh * u * da, dh * a}, -1);
      const auto type = v[0].scalar_type();
      if (need_x) out[0] = at::matmul(dgu, w13).to(type);
      if (need_w13) out[1] = at::matmul(rows2d(dgu).t(), rows2d(x)).to(type);
      if (need_w2) out[2] = at::matmul(rows2d(d).t(), rows2d(a * u)).to(type);
    } else if (need_x || need_w13 || need_w2) {
      auto [dx, dw13, dw2] = gated_ffn_bwd(rows2d(dy), rows2d(v[0]), v[1], v[2], opt(v[3]), opt(v[4]),
                                           ctx->saved_data["act"].toInt(), need_x, need_w13, need_w2);
      if (dx) out[0] = dx->view(v[0].sizes());
      out[1] = val(dw13);
      out[2] = val(dw2);
    }
    if (ctx->saved_data["residual"].toBool()) out[3] = dy;
    return out;
  }
};

// The block, or None where the kernels do not cover the type, the sizes or the kind of tensor (the caller's plain form does)
OptT gated_ffn(const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w2, const OptT& residual, int64_t act) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && w13.dim() == 2 && w2.dim() == 2 && w13.size(1) == x.size(-1) &&
                        w13.size(0) == 2 * w2.size(1),
                    "gated_ffn: x [..., H], w13 [2F, H], w2 [N, F]; got ", x.sizes(), ", ", w13.sizes(), ", ",
                    w2.sizes());
  TORCH_CHECK_VALUE(w13.numel() > 0 && w2.numel() > 0, "gated_ffn: empty feature dimension");
  for (const at::Tensor* t : {&w13, &w2, residual ? &*residual : &w2})
    TORCH_CHECK_VALUE(t->device() == x.device() && t->scalar_type() == x.scalar_type(),
                      "gated_ffn: weights and residual have x's type and device");
  if (residual) {
    TORCH_CHECK_VALUE(residual->dim() == x.dim() && residual->size(-1) == w2.size(0) &&
                          residual->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
                      "gated_ffn: residual [..., N] with x's leading dimensions");
  }
  const bool half = x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf;
  if (!x.is_cuda() || !half || x.size(-1) % 8 || w2.size(0) % 8 || w2.size(1) % 8) return OptT();
  if (!launchable(x, w13, w2, residual)) return OptT();
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w13) || wants_grad(w2) || wants_grad(residual)))
    return GatedFfn::apply(x, w13, w2, residual, act);
  return std::get<0>(gated_ffn_fwd(x, w13, w2, residual, act, false));
}

struct TrainNorm : torch::autograd::Function<TrainNorm> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const OptT& b, double eps,
                            bool rms) {
    const at::Tensor wc = w.contiguous();
    auto [y, mean, rstd] = norm_train_fwd(x, wc, b ? OptT(b->contiguous()) : OptT(), eps, rms, true);
    ctx->save_for_backward({x, w, val(mean), val(rstd)});
    ctx->saved_data["rms"] = rms;
    ctx->saved_data["bias"] = b.has_value();
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool rms = ctx->saved_data["rms"].toBool(), need_x = ctx->needs_input_grad(0),
               need_w = ctx->needs_input_grad(1),
               need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    capturable_backward(rms ? "rms_norm" : "layer_norm");
    const variable_list v = ctx->get_saved_variables();
    variable_list out(5);
    // create_graph, or gradients that no kernel can take: the formulas in operations that can be differentiated again
    if (at::GradMode::is_enabled() || !launchable(grads[0])) {
      const at::Tensor x = v[0].to(at::kFloat), w = v[1].to(at::kFloat), dy = grads[0].to(at::kFloat);
      const at::Tensor c = rms ? x : x - x.mean({-1}, true);
      const at::Tensor rstd = at::rsqrt(c.square().mean({-1}, true) + ctx->saved_data["eps"].toDouble());
      const at::Tensor xh = c * rstd, g = dy * (rms ? 1. + w : w);
      at::Tensor d = g - xh * (g * xh).mean({-1}, true);
      if (!rms) d = d - g.mean({-1}, true);
      if (need_x) out[0] = (rstd * d).to(v[0].scalar_type());
      if (need_w) out[1] = rows2d(dy * xh).sum(0).to(v[1].scalar_type());
      if (need_b) out[2] = rows2d(dy).sum(0).to(v[1].scalar_type());
      return out;
    }
    auto [dx, dw, db] = norm_train_bwd(rows2d(grads[0]), norm_rows(v[0]), v[1].contiguous(), opt(v[2]), v[3], rms,
                                       need_x, need_w, need_b);
    if (dx) out[0] = dx->view(v[0].sizes());
    out[1] = val(dw);
    out[2] = val(db);
    return out;
  }
};

// The norm, or None for tensors that the kernels cannot read (the caller's plain form does)
OptT train_norm(const at::Tensor& x, const at::Tensor& w, const OptT& b, double eps, bool rms) {
  if (!launchable(x, w, b)) return OptT();
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "norm: x [..., width]");
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b)))
    return TrainNorm::apply(x, w, b, eps, rms);
  return std::get<0>(norm_train_fwd(x, w.contiguous(), b ? OptT(b->contiguous()) : OptT(), eps, rms, false));
}

struct Dropout : torch::autograd::Function<Dropout> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptT& residual, const OptT& rng,
                            int64_t threshold, int64_t seed, int64_t offset) {
    ctx->save_for_backward({val(rng)});
    ctx->saved_data["threshold"] = threshold;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["residual"] = residual.has_value();
    return dropout_op(x, residual, threshold, seed, offset, rng);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    differentiable_once("dropout");
    capturable_backward("dropout");
    variable_list out(6);
    if (ctx->needs_input_grad(0)) {
      const int64_t threshold = ctx->saved_data["threshold"].toInt();
      auto masked = [&](const at::Tensor& t) {
        return dropout_op(t, OptT(), threshold, ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt(),
                          opt(ctx->get_saved_variables()[0]));
      };
      const at::Tensor& dy = grads[0];
      if (launchable(dy)) {
        out[0] = masked(dy);
      } else {  // the mask from a tensor that no transform and no mode knows of
        at::Tensor keep;
        {
          c10::impl::ExcludeDispatchKeyGuard unseen(
              c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::Tracer,
                                   c10::DispatchKey::FuncTorchDynamicLayerFrontMode,
                                   c10::DispatchKey::FuncTorchDynamicLayerBackMode}));
          const auto device = at::TensorOptions().dtype(at::kFloat).device(dy.device());
          keep = masked(at::ones(dy.sizes(), device)).ne(0.);
        }
        const at::Tensor y = dy.to(at::kFloat) * (threshold ? 65536. / threshold : 0.);
        out[0] = at::where(keep, y, at::zeros({}, y.options())).to(dy.scalar_type());
      }
    }
    if (ctx->saved_data["residual"].toBool()) out[1] = grads[0];
    return out;
  }
};

// y, or None for tensors that the kernel cannot read
OptT dropout(const at::Tensor& x, const OptT& residual, int64_t threshold, int64_t seed, int64_t offset,
             const OptT& rng) {
  if (!launchable(x, residual, rng)) return OptT();
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(residual)))
    return Dropout::apply(x, residual, rng, threshold, seed, offset);
  return dropout_op(x, residual, threshold, seed, offset, rng);
}

}  // namespace

void register_ffn(pybind11::module& m) {
  m.def("gated_ffn", &gated_ffn, py::arg("x"), py::arg("w13"), py::arg("w2"), py::arg("residual"), py::arg("act"));
  m.def("train_norm", &train_norm, py::arg("x"), py::arg("w"), py::arg("b"), py::arg("eps"), py::arg("rms"));
  m.def("dropout", &dropout, py::arg("x"), py::arg("residual"), py::arg("threshold"), py::arg("seed"),
        py::arg("offset"), py::arg("rng"));
}
