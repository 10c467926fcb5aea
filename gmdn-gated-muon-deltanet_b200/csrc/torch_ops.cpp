// torch operators over the C ABI for the training step's kernels (norm, token
// log probabilities, 8-bit activations), registered as gmdn::* with their
// autograd formulas; built into libgmdn_torch.so, which links libgmdn_b200.so.
//
// They are in C++ because the kernels of a small call take a few microseconds:
// the same ops written in Python cost 140 us of host time for one norm forward
// and backward, more than the same norm in elementary torch operations.
//
// Every op takes tensors of any strides (it copies what its kernel cannot read
// in place), runs on the current stream of the tensors' device, and checks what
// its kernel relies on: devices, types and shapes.  Fake kernels are registered
// from Python (step_ops.py).

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <initializer_list>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/gmdn_scan.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kBlock8 = 128;   // elements that share a scale

void check(int rc, const char* what) {
  TORCH_CHECK(rc == GMDN_OK, what, " failed (code ", rc, "): ", gmdn_last_error_string());
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
bool is_f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }

// What a kernel may be given: contiguous and aligned (a copy where t is not).
Tensor dense(const Tensor& t, uintptr_t align = 16) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % align ? c.clone() : c;
}
OptTensor dense(const OptTensor& t, uintptr_t align = 16) {
  return has(t) ? OptTensor(dense(*t, align)) : OptTensor();
}
template <typename T = void>
const T* in(const OptTensor& t) {
  return has(t) ? static_cast<const T*>(t->const_data_ptr()) : nullptr;
}
template <typename T = void>
T* out(Tensor& t) {   // an output that was not asked for is empty
  return t.numel() ? static_cast<T*>(t.mutable_data_ptr()) : nullptr;
}

void check_act(const Tensor& t, const char* what) {
  const auto s = t.scalar_type();
  TORCH_CHECK_TYPE(s == at::kBFloat16 || s == at::kFloat, what,
                   " must be bfloat16 or float32, got ", s);
}
void check_like(const char* op, const Tensor& first, const OptTensor& t) {
  TORCH_CHECK(!has(t) || t->device() == first.device(), op, ": tensors on ", first.device(),
              " and ", t->device());
}
void check_f32(const char* op, const OptTensor& t, int64_t n) {
  TORCH_CHECK(!has(t) || (is_f32(*t) && t->numel() == n), op, ": expected ", n,
              " float32 values");
}
// A forward-mode tangent: it needs neither requires_grad nor grad mode.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
// Whether autograd has anything to record, or a tangent to refuse (there is no forward mode, and
// autograd's path says so).
bool any_derivative(std::initializer_list<const Tensor*> ts,
                    std::initializer_list<const OptTensor*> opts) {
  const bool grad = c10::GradMode::is_enabled();
  auto wants = [grad](const Tensor& t) { return (grad && t.requires_grad()) || has_tangent(t); };
  for (const Tensor* t : ts)
    if (wants(*t)) return true;
  for (const OptTensor* t : opts)
    if (has(*t) && wants(**t)) return true;
  return false;
}
// In a plain backward (grad mode off, cotangents without tangents) its op goes straight to the
// kernel, past the boxed fallback that refuses second derivatives and tangents.
struct BelowAutograd {
  std::optional<at::AutoDispatchBelowADInplaceOrView> guard;
  explicit BelowAutograd(const variable_list& cotangents) {
    if (c10::GradMode::is_enabled()) return;
    for (const Tensor& t : cotangents)
      if (has_tangent(t)) return;
    guard.emplace();
  }
};
void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}
at::TensorOptions f32_like(const Tensor& t) { return t.options().dtype(at::kFloat); }

// ---------------------------------------------------------------------------
// norm
// ---------------------------------------------------------------------------

using Norm = std::tuple<Tensor, Tensor, Tensor>;                 // y, h, stats
using NormGrads = std::tuple<Tensor, Tensor, Tensor, Tensor>;    // bf16 ds, fp32 ds, dw, db

Norm norm_fwd_cuda(const Tensor& x0, const OptTensor& res0, const OptTensor& w0,
                   const OptTensor& b0, double eps, bool center, bool out_f32) {
  check_act(x0, "x");
  TORCH_CHECK(x0.dim() >= 1, "norm: x must have a last axis");
  const int64_t D = x0.size(-1), rows = D ? x0.numel() / D : 0;
  TORCH_CHECK(D < (1ll << 31), "norm: width ", D, " is too large");
  for (const OptTensor* t : {&res0, &w0, &b0}) check_like("norm", x0, *t);
  check_f32("norm", w0, D);
  check_f32("norm", b0, D);
  if (has(res0)) {
    check_act(*res0, "residual");
    TORCH_CHECK(res0->sizes() == x0.sizes(), "norm: residual and x differ in shape");
  }
  const c10::cuda::CUDAGuard guard(x0.device());
  const Tensor x = dense(x0);
  const OptTensor res = dense(res0), w = dense(w0), b = dense(b0);
  const bool h_f32 = is_f32(x) || (has(res) && is_f32(*res));
  Tensor y = at::empty(x.sizes(), x.options().dtype(out_f32 ? at::kFloat : at::kBFloat16));
  Tensor h = has(res) ? at::empty(x.sizes(), x.options().dtype(h_f32 ? at::kFloat : at::kBFloat16))
                      : at::empty({0}, x.options());
  Tensor stats = at::empty({center ? 2 : 1, rows}, f32_like(x));
  float* st = static_cast<float*>(stats.mutable_data_ptr());
  check(gmdn_norm_fwd(x.const_data_ptr(), in(res), in<float>(w), in<float>(b),
                      y.mutable_data_ptr(), out(h), st, center ? st + rows : nullptr, rows,
                      static_cast<int>(D), static_cast<float>(eps), center, is_f32(x),
                      has(res) && is_f32(*res), out_f32, stream_of(x)),
        "gmdn_norm_fwd");
  return {y, h, stats};
}

NormGrads norm_bwd_cuda(const Tensor& s0, const Tensor& stats0, const OptTensor& w0,
                        const Tensor& dy0, const OptTensor& dh0, bool center, bool want_bf16,
                        bool want_f32, bool want_w, bool want_b) {
  check_act(s0, "s");
  check_act(dy0, "dy");
  const int64_t D = s0.size(-1), rows = D ? s0.numel() / D : 0;
  check_like("norm", s0, stats0);
  check_like("norm", s0, w0);
  check_like("norm", s0, dy0);
  check_like("norm", s0, dh0);
  check_f32("norm", stats0, (center ? 2 : 1) * rows);
  check_f32("norm", w0, D);
  TORCH_CHECK(dy0.sizes() == s0.sizes(), "norm: dy and s differ in shape");
  TORCH_CHECK(!has(dh0) || (dh0->sizes() == s0.sizes() && dh0->scalar_type() == s0.scalar_type()),
              "norm: dh must be like h");
  const c10::cuda::CUDAGuard guard(s0.device());
  const Tensor s = dense(s0), stats = stats0.contiguous(), dy = dense(dy0);
  const OptTensor w = dense(w0), dh = dense(dh0);
  auto make = [&](bool wanted, at::IntArrayRef shape, at::ScalarType type) {
    return wanted ? at::empty(shape, s.options().dtype(type))
                  : at::empty({0}, s.options().dtype(type));
  };
  Tensor da = make(want_bf16, s.sizes(), at::kBFloat16);
  Tensor db = make(want_f32, s.sizes(), at::kFloat);
  Tensor dw = make(want_w, {D}, at::kFloat), dbias = make(want_b, {D}, at::kFloat);
  const size_t need =
      want_w || want_b ? gmdn_norm_bwd_workspace_bytes(rows, static_cast<int>(D)) : 0;
  Tensor ws = need ? at::empty({static_cast<int64_t>(need)}, s.options().dtype(at::kByte)) : Tensor();
  const float* st = static_cast<const float*>(stats.const_data_ptr());
  check(gmdn_norm_bwd(s.const_data_ptr(), st, center ? st + rows : nullptr, in<float>(w),
                      dy.const_data_ptr(), in(dh), out(da), out(db), out<float>(dw),
                      out<float>(dbias), need ? ws.mutable_data_ptr() : nullptr, need, rows,
                      static_cast<int>(D), center, is_f32(s), is_f32(dy), has(dh) && is_f32(*dh), 0,
                      1, stream_of(s)),
        "gmdn_norm_bwd");
  return {da, db, dw, dbias};
}

Norm norm_fwd_op(const Tensor& x, const OptTensor& res, const OptTensor& w, const OptTensor& b,
                 double eps, bool center, bool out_f32) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("gmdn::norm_fwd", "")
                       .typed<decltype(norm_fwd_cuda)>();
  return op.call(x, res, w, b, eps, center, out_f32);
}
NormGrads norm_bwd_op(const Tensor& s, const Tensor& stats, const OptTensor& w, const Tensor& dy,
                      const OptTensor& dh, bool center, bool a, bool b, bool c, bool d) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("gmdn::norm_bwd", "")
                       .typed<decltype(norm_bwd_cuda)>();
  return op.call(s, stats, w, dy, dh, center, a, b, c, d);
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  // one saved word: the map of saved data costs more than the values
  enum : int64_t { kCenter = 1, kOutF32 = 2, kXF32 = 4, kRes = 8, kResF32 = 16, kNeedX = 32,
                   kNeedRes = 64, kNeedW = 128, kNeedB = 256 };
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& res,
                               const OptTensor& w, const OptTensor& b, double eps, bool center,
                               bool out_f32) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, h, stats] = norm_fwd_op(x, res, w, b, eps, center, out_f32);
    auto wants = [](const OptTensor& t) { return has(t) && t->requires_grad(); };
    const int64_t flags = (center ? kCenter : 0) | (out_f32 ? kOutF32 : 0) |
                          (is_f32(x) ? kXF32 : 0) | (has(res) ? kRes : 0) |
                          (has(res) && is_f32(*res) ? kResF32 : 0) |
                          (x.requires_grad() ? kNeedX : 0) | (wants(res) ? kNeedRes : 0) |
                          (wants(w) ? kNeedW : 0) | (wants(b) ? kNeedB : 0);
    ctx->saved_data["flags"] = flags;
    ctx->save_for_backward({has(res) ? h : x, stats, has(w) ? *w : Tensor()});
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable(has(res) ? variable_list{stats} : variable_list{h, stats});
    return {y, h, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    auto flag = [flags](int64_t f) { return (flags & f) != 0; };
    const Tensor &s = saved[0], &w = saved[2];
    const bool res = flag(kRes), x_f32 = flag(kXF32), res_f32 = flag(kResF32);
    const OptTensor dh = res && grads[1].defined() ? OptTensor(grads[1]) : OptTensor();
    const bool need_x = flag(kNeedX), need_res = flag(kNeedRes);
    if (!grads[0].defined()) {
      // y is not used: the cotangent of h alone (the formula would make NaN of 0 times a row
      // that holds an infinity)
      auto as = [&](bool need, bool f32) {
        return need && has(dh) ? dh->to(f32 ? at::kFloat : at::kBFloat16) : Tensor();
      };
      auto none = [&](int64_t f) {
        return flag(f) ? at::zeros({s.size(-1)}, f32_like(s)) : Tensor();
      };
      return {as(need_x, x_f32), as(need_res, res_f32), none(kNeedW), none(kNeedB),
              Tensor(), Tensor(), Tensor()};
    }
    const Tensor dy = grads[0].to(flag(kOutF32) ? at::kFloat : at::kBFloat16);
    const BelowAutograd below(grads);
    auto [da, db, dw, dbias] =
        norm_bwd_op(s, saved[1], w.defined() ? OptTensor(w) : OptTensor(), dy, dh, flag(kCenter),
                    (need_x && !x_f32) || (need_res && !res_f32),
                    (need_x && x_f32) || (need_res && res_f32), flag(kNeedW), flag(kNeedB));
    return {need_x ? (x_f32 ? db : da) : Tensor(), need_res ? (res_f32 ? db : da) : Tensor(),
            flag(kNeedW) ? dw : Tensor(), flag(kNeedB) ? dbias : Tensor(),
            Tensor(), Tensor(), Tensor()};
  }
};

Norm norm_fwd_autograd(const Tensor& x, const OptTensor& res, const OptTensor& w,
                       const OptTensor& b, double eps, bool center, bool out_f32) {
  if (!any_derivative({&x}, {&res, &w, &b})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return norm_fwd_op(x, res, w, b, eps, center, out_f32);
  }
  auto r = NormFunction::apply(x, res, w, b, eps, center, out_f32);
  return {r[0], r[1], r[2]};
}

// ---------------------------------------------------------------------------
// token log probabilities
// ---------------------------------------------------------------------------

// logprobs, entropy, top logprobs, top ids, stats
using Logprobs = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

// Rows of a tensor whose rows are contiguous as (batch, length) with two
// strides; false where two strides do not reach every row.
struct Rows {
  int64_t batch = 1, length = 1, stride_b = 0, stride_t = 0;
  bool from(const Tensor& t) {
    const int64_t n = t.dim() - 1;
    if (t.numel() == 0) {
      batch = length = 0;
      return true;
    }
    if (t.size(n) > 1 && t.stride(n) != 1) return false;
    batch = length = 1;
    stride_b = stride_t = 0;
    int parts = 0;
    for (int64_t d = 0; d < n; ++d) {
      if (t.size(d) == 1) continue;
      if (parts && stride_t == t.size(d) * t.stride(d)) {
        length *= t.size(d);
        stride_t = t.stride(d);
        continue;
      }
      if (++parts > 2) return false;
      batch = length;
      stride_b = stride_t;
      length = t.size(d);
      stride_t = t.stride(d);
    }
    return true;
  }
};

void check_logits(const Tensor& logits, const OptTensor& targets) {
  check_act(logits, "logits");
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) < (1ll << 31),
              "token_logprobs: logits must be (..., V)");
  check_like("token_logprobs", logits, targets);
  if (has(targets)) {
    TORCH_CHECK(targets->scalar_type() == at::kLong, "token_logprobs: targets must be int64");
    TORCH_CHECK(targets->sizes() == logits.sizes().slice(0, logits.dim() - 1),
                "token_logprobs: targets do not fit the logits");
  }
}

Logprobs token_logprobs_fwd_cuda(const Tensor& logits0, const OptTensor& targets0, bool entropy,
                                 int64_t top_k, int64_t ignore_index) {
  check_logits(logits0, targets0);
  const c10::cuda::CUDAGuard guard(logits0.device());
  Tensor logits = logits0;
  Rows rows;
  if (!rows.from(logits)) {
    logits = logits.contiguous();
    rows.from(logits);
  }
  const OptTensor targets = has(targets0) ? OptTensor(targets0->contiguous()) : OptTensor();
  const auto shape = logits.sizes().slice(0, logits.dim() - 1).vec();
  const auto opts = f32_like(logits);
  auto with = [&](int64_t n) {
    auto s = shape;
    s.push_back(n);
    return s;
  };
  const std::vector<int64_t> none{0};
  Tensor stats = at::empty(with(4), opts);
  Tensor lp = at::empty(has(targets) ? shape : none, opts);
  Tensor ent = at::empty(entropy ? shape : none, opts);
  Tensor tops = at::empty(top_k ? with(top_k) : none, opts);
  Tensor ids = at::empty(top_k ? with(top_k) : none, opts.dtype(at::kLong));
  check(gmdn_token_logprobs_fwd(
            logits.const_data_ptr(), in<int64_t>(targets), has(targets) ? out<float>(lp) : nullptr,
            entropy ? out<float>(ent) : nullptr, out<float>(tops), out<int64_t>(ids),
            out<float>(stats), rows.batch, rows.length, rows.stride_b, rows.stride_t,
            static_cast<int>(logits.size(-1)), static_cast<int>(top_k), ignore_index,
            is_f32(logits), stream_of(logits)),
        "gmdn_token_logprobs_fwd");
  return {lp, ent, tops, ids, stats};
}

Tensor token_logprobs_bwd_cuda(const Tensor& logits0, const OptTensor& targets0,
                               const OptTensor& ids0, const Tensor& stats0, const OptTensor& g_lp0,
                               const OptTensor& g_ent0, const OptTensor& g_top0,
                               int64_t ignore_index) {
  check_logits(logits0, targets0);
  const int64_t V = logits0.size(-1), n = logits0.numel() / V;
  for (const OptTensor* t : {&ids0, &g_lp0, &g_ent0, &g_top0})
    check_like("token_logprobs", logits0, *t);
  check_like("token_logprobs", logits0, stats0);
  check_f32("token_logprobs", stats0, 4 * n);
  check_f32("token_logprobs", g_lp0, n);
  check_f32("token_logprobs", g_ent0, n);
  TORCH_CHECK(!has(g_lp0) || has(targets0), "token_logprobs: g_logprobs without targets");
  const int64_t k = has(g_top0) ? g_top0->size(-1) : 0;
  if (k) {
    TORCH_CHECK(has(ids0) && ids0->scalar_type() == at::kLong && ids0->sizes() == g_top0->sizes(),
                "token_logprobs: g_top and top_ids differ");
    check_f32("token_logprobs", g_top0, n * k);
  }
  const c10::cuda::CUDAGuard guard(logits0.device());
  Tensor logits = logits0;
  Rows rows;
  if (!rows.from(logits)) {
    logits = logits.contiguous();
    rows.from(logits);
  }
  auto flat = [](const OptTensor& t) { return has(t) ? OptTensor(t->contiguous()) : OptTensor(); };
  const OptTensor targets = flat(targets0), ids = flat(ids0), g_lp = flat(g_lp0),
                  g_ent = flat(g_ent0), g_top = k ? flat(g_top0) : OptTensor();
  const Tensor stats = dense(stats0);
  Tensor grad = at::empty(logits.sizes(), logits.options());
  check(gmdn_token_logprobs_bwd(logits.const_data_ptr(), in<int64_t>(targets),
                                static_cast<const float*>(stats.const_data_ptr()),
                                in<int64_t>(ids), in<float>(g_lp), in<float>(g_ent),
                                in<float>(g_top), grad.mutable_data_ptr(), rows.batch, rows.length,
                                rows.stride_b, rows.stride_t, static_cast<int>(V),
                                static_cast<int>(k), ignore_index, is_f32(logits),
                                stream_of(logits)),
        "gmdn_token_logprobs_bwd");
  return grad;
}

Logprobs token_logprobs_fwd_op(const Tensor& logits, const OptTensor& targets, bool entropy,
                               int64_t top_k, int64_t ignore_index) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("gmdn::token_logprobs_fwd", "")
                       .typed<decltype(token_logprobs_fwd_cuda)>();
  return op.call(logits, targets, entropy, top_k, ignore_index);
}
Tensor token_logprobs_bwd_op(const Tensor& logits, const OptTensor& targets, const OptTensor& ids,
                             const Tensor& stats, const OptTensor& g_lp, const OptTensor& g_ent,
                             const OptTensor& g_top, int64_t ignore_index) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("gmdn::token_logprobs_bwd", "")
                       .typed<decltype(token_logprobs_bwd_cuda)>();
  return op.call(logits, targets, ids, stats, g_lp, g_ent, g_top, ignore_index);
}

struct LogprobsFunction : torch::autograd::Function<LogprobsFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& targets,
                               bool entropy, int64_t top_k, int64_t ignore_index) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [lp, ent, tops, ids, stats] =
        token_logprobs_fwd_op(logits, targets, entropy, top_k, ignore_index);
    ctx->saved_data["ignore"] = ignore_index;
    ctx->saved_data["entropy"] = entropy;
    ctx->saved_data["top_k"] = top_k;
    ctx->save_for_backward(
        {logits, has(targets) ? *targets : Tensor(), top_k ? ids : Tensor(), stats});
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({ids, stats});
    return {lp, ent, tops, ids, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    auto cot = [&](int i, bool used) {
      return used && grads[i].defined() ? OptTensor(grads[i].to(at::kFloat)) : OptTensor();
    };
    const BelowAutograd below(grads);
    Tensor g = token_logprobs_bwd_op(
        saved[0], opt(saved[1]), opt(saved[2]), saved[3], cot(0, saved[1].defined()),
        cot(1, ctx->saved_data["entropy"].toBool()), cot(2, ctx->saved_data["top_k"].toInt() > 0),
        ctx->saved_data["ignore"].toInt());
    return {g, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Logprobs token_logprobs_fwd_autograd(const Tensor& logits, const OptTensor& targets, bool entropy,
                                     int64_t top_k, int64_t ignore_index) {
  if (!any_derivative({&logits}, {})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return token_logprobs_fwd_op(logits, targets, entropy, top_k, ignore_index);
  }
  auto r = LogprobsFunction::apply(logits, targets, entropy, top_k, ignore_index);
  return {r[0], r[1], r[2], r[3], r[4]};
}

// ---------------------------------------------------------------------------
// activations in 8 bits
// ---------------------------------------------------------------------------

constexpr uintptr_t kAlign8 = 32;

std::pair<Tensor, Tensor> codes_like(const Tensor& x) {
  return {at::empty(x.sizes(), x.options().dtype(at::kChar)),
          at::empty({(x.numel() + kBlock8 - 1) / kBlock8}, f32_like(x))};
}
void check_codes(const char* op, const Tensor& codes, const Tensor& scales) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kChar && is_f32(scales), op,
                   ": codes must be int8 and scales float32");
  TORCH_CHECK_VALUE(scales.numel() == (codes.numel() + kBlock8 - 1) / kBlock8, op,
                    ": one scale for each 128 codes");
  check_like(op, codes, scales);
}
const int8_t* i8(const Tensor& t) { return static_cast<const int8_t*>(t.const_data_ptr()); }
const float* f32(const Tensor& t) { return static_cast<const float*>(t.const_data_ptr()); }

std::tuple<Tensor, Tensor> pack8_cuda(const Tensor& x0) {
  check_act(x0, "x");
  const c10::cuda::CUDAGuard guard(x0.device());
  const Tensor x = dense(x0, kAlign8);
  auto [codes, scales] = codes_like(x);
  check(gmdn_pack8(x.const_data_ptr(), out<int8_t>(codes), out<float>(scales), x.numel(), is_f32(x),
                   stream_of(x)),
        "gmdn_pack8");
  return {codes, scales};
}

Tensor unpack8_cuda(const Tensor& codes0, const Tensor& scales0, bool to_f32) {
  check_codes("unpack8", codes0, scales0);
  const c10::cuda::CUDAGuard guard(codes0.device());
  const Tensor codes = dense(codes0, kAlign8), scales = dense(scales0, kAlign8);
  Tensor x = at::empty(codes.sizes(), codes.options().dtype(to_f32 ? at::kFloat : at::kBFloat16));
  check(gmdn_unpack8(i8(codes), f32(scales), out(x), x.numel(), to_f32, stream_of(x)),
        "gmdn_unpack8");
  return x;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> act8_fwd_cuda(const Tensor& x0,
                                                                 const OptTensor& gate0) {
  check_act(x0, "x");
  check_like("act8", x0, gate0);
  TORCH_CHECK(!has(gate0) || (gate0->sizes() == x0.sizes() &&
                              gate0->scalar_type() == x0.scalar_type()),
              "act8: the gate must be like x");
  const c10::cuda::CUDAGuard guard(x0.device());
  const Tensor x = dense(x0, kAlign8);
  const OptTensor gate = dense(gate0, kAlign8);
  Tensor y = at::empty(x.sizes(), x.options());
  auto [codes, scales] = codes_like(x);
  Tensor gcodes, gscales;
  if (has(gate)) {
    std::tie(gcodes, gscales) = codes_like(x);
  } else {
    gcodes = at::empty({0}, codes.options());
    gscales = at::empty({0}, scales.options());
  }
  check(gmdn_act8_fwd(x.const_data_ptr(), in(gate), out(y), out<int8_t>(codes), out<float>(scales),
                      out<int8_t>(gcodes), out<float>(gscales), x.numel(), is_f32(x),
                      stream_of(x)),
        "gmdn_act8_fwd");
  return {y, codes, scales, gcodes, gscales};
}

std::tuple<Tensor, Tensor, Tensor> act8_bwd_cuda(const Tensor& codes0, const Tensor& scales0,
                                                 const OptTensor& gcodes0,
                                                 const OptTensor& gscales0, const Tensor& dy0,
                                                 bool restore) {
  check_act(dy0, "dy");
  check_codes("act8", codes0, scales0);
  check_like("act8", dy0, codes0);
  TORCH_CHECK(dy0.sizes() == codes0.sizes(), "act8: dy and the checkpoint differ in shape");
  TORCH_CHECK(has(gcodes0) == has(gscales0), "act8: a gate's codes need its scales");
  if (has(gcodes0)) {
    check_codes("act8", *gcodes0, *gscales0);
    check_like("act8", dy0, gcodes0);
    TORCH_CHECK(gcodes0->sizes() == codes0.sizes(), "act8: the gate's checkpoint differs in shape");
  }
  const c10::cuda::CUDAGuard guard(dy0.device());
  const Tensor codes = dense(codes0, kAlign8), scales = dense(scales0, kAlign8),
               dy = dense(dy0, kAlign8);
  const OptTensor gcodes = dense(gcodes0, kAlign8), gscales = dense(gscales0, kAlign8);
  Tensor dx = at::empty(dy.sizes(), dy.options());
  Tensor dgate = has(gcodes) ? at::empty(dy.sizes(), dy.options()) : at::empty({0}, dy.options());
  Tensor y = restore ? at::empty(dy.sizes(), dy.options()) : at::empty({0}, dy.options());
  check(gmdn_act8_bwd(i8(codes), f32(scales), in<int8_t>(gcodes), in<float>(gscales),
                      dy.const_data_ptr(), out(dx), out(dgate), out(y), dy.numel(), is_f32(dy),
                      stream_of(dy)),
        "gmdn_act8_bwd");
  return {dx, dgate, y};
}

TORCH_LIBRARY_FRAGMENT(gmdn, m) {
  m.def("norm_fwd(Tensor x, Tensor? residual, Tensor? weight, Tensor? bias, float eps, bool center, "
        "bool out_f32) -> (Tensor, Tensor, Tensor)");
  m.def("norm_bwd(Tensor s, Tensor stats, Tensor? weight, Tensor dy, Tensor? dh, bool center, "
        "bool want_bf16, bool want_f32, bool want_w, bool want_b) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("token_logprobs_fwd(Tensor logits, Tensor? targets, bool entropy, int top_k, "
        "int ignore_index) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("token_logprobs_bwd(Tensor logits, Tensor? targets, Tensor? ids, Tensor stats, "
        "Tensor? g_lp, Tensor? g_ent, Tensor? g_top, int ignore_index) -> Tensor");
  m.def("pack8(Tensor x) -> (Tensor, Tensor)");
  m.def("unpack8(Tensor codes, Tensor scales, bool f32) -> Tensor");
  m.def("act8_fwd(Tensor x, Tensor? gate) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("act8_bwd(Tensor codes, Tensor scales, Tensor? gcodes, Tensor? gscales, Tensor dy, "
        "bool restore) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(gmdn, CUDA, m) {
  m.impl("norm_fwd", norm_fwd_cuda);
  m.impl("norm_bwd", norm_bwd_cuda);
  m.impl("token_logprobs_fwd", token_logprobs_fwd_cuda);
  m.impl("token_logprobs_bwd", token_logprobs_bwd_cuda);
  m.impl("pack8", pack8_cuda);
  m.impl("unpack8", unpack8_cuda);
  m.impl("act8_fwd", act8_fwd_cuda);
  m.impl("act8_bwd", act8_bwd_cuda);
}

TORCH_LIBRARY_IMPL(gmdn, Autograd, m) {
  m.impl("norm_fwd", norm_fwd_autograd);
  m.impl("token_logprobs_fwd", token_logprobs_fwd_autograd);
  // no derivative: a second one through these raises
  for (const char* name : {"norm_bwd", "token_logprobs_bwd"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
  // checkpoints: autograd does not see them
  for (const char* name : {"pack8", "unpack8", "act8_fwd", "act8_bwd"})
    m.impl(name, torch::CppFunction::makeFallthrough());
}

}  // namespace
