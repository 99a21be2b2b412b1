// Python binding of single operators of liblmufft_hip.so: their checks, outputs, workspaces and autograd functions.
//
// A frame of a stream is a few microseconds of kernel; argument checks, tensor bookkeeping and an autograd function written
// in Python cost several times that a call (measured: a step of four streams 14.3 us a call, a training pass of the smallest
// utterances 143 us, of which 48 us are torch's own).  The C ABI (include/lmufft.h) stays the library's boundary: this file
// calls nothing else of it, through addresses that asr_amd/_call.py hands over, so that the same library is used that ctypes
// has loaded.
#include <ATen/autocast_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <string>
#include <unordered_map>

#include "lmufft.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

// ---- the library's entry points
#define LMUFFT_ENTRIES(X)                                                                                       \
  X(lmufft_last_error) X(lmufft_decay_workspace_bytes) X(lmufft_decay_attention) X(lmufft_decay_attention_bwd)   \
  X(lmufft_decay_attention_step) X(lmufft_group_norm_workspace_bytes) X(lmufft_group_norm) X(lmufft_group_norm_bwd) \
  X(lmufft_dropout_add)
struct Library {
#define X(name) decltype(&::name) name = nullptr;
  LMUFFT_ENTRIES(X)
#undef X
} lib;

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
#define X(name) lib.name = reinterpret_cast<decltype(lib.name)>(at.at(#name));
  LMUFFT_ENTRIES(X)
#undef X
}

void ran(int rc, const char* what) { TORCH_CHECK(rc == 0, what, ": ", lib.lmufft_last_error()); }

// ---- what every operator needs
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? LMUFFT_F32 : LMUFFT_BF16; }
bool known(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
template <class T>
T* ptr_mut(const Tensor& t) { return t.defined() ? static_cast<T*>(t.mutable_data_ptr()) : nullptr; }

struct OnDevice {  // the device of a call made current for it, and its stream there
  explicit OnDevice(const Tensor& t)
      : guard(t.device()), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream()) {}
  c10::OptionalDeviceGuard guard;
  void* stream;
};

void on_gpu(const char* what, const char* name, const Tensor& t, const Tensor& like, const char* like_name) {
  TORCH_CHECK(t.is_cuda(), what, ": `", name, "` lives on ", t.device(),
              "; the kernels run only on a GPU (there is no CPU fallback)");
  TORCH_CHECK(t.device() == like.device(), what, ": `", name, "` lives on ", t.device(), ", ", like_name, " on ", like.device());
}

// `t` contiguous from a 16-byte boundary on
Tensor dense(const Tensor& t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 == 0 ? c : c.clone();
}

// `counts` [batch] (frames of each utterance, or which streams are live) as the kernels read it
Tensor frames_of(const char* what, const char* name, const MaybeTensor& counts, const Tensor& like, int64_t batch) {
  if (!counts.has_value() || !counts->defined()) return Tensor();
  TORCH_CHECK(counts->dim() == 1 && counts->size(0) == batch, what, ": `", name, "` must have shape (", batch, ",), got ", counts->sizes());
  TORCH_CHECK(!counts->is_floating_point() && !counts->is_complex(), what, ": `", name, "` must hold whole numbers, got ", counts->scalar_type());
  // what does not fit 32 bits keeps its meaning
  const Tensor fit = counts->scalar_type() == at::kLong ? counts->clamp(0, INT32_MAX) : *counts;
  return fit.to(like.device(), at::kInt).contiguous();
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}

// The gradients of a backward that has no backward of its own.
variable_list once(const char* what, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  const auto n = (int64_t)grads.size();
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": the backward is not differentiable", n);
  return (*error)(std::move(grads));
}

// ---- causal decay attention (asr_amd/decay.py)
struct Rows {  // a [B][T][width] tensor with rows the kernels can load 16 bytes at a time
  const void* p;
  int64_t ld, bs;
};
bool rows_fit(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  return t.stride(2) == 1 && (t.size(1) == 1 || (t.stride(1) % per == 0 && t.stride(1) <= 1 << 22)) && (t.size(0) == 1 || t.stride(0) % per == 0) &&
         reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}
Tensor with_rows(const Tensor& t) { return t.numel() == 0 || rows_fit(t) ? t : dense(t); }
Rows rows_of(const Tensor& t, int64_t first_column = 0) {
  return {static_cast<const char*>(t.const_data_ptr()) + first_column * t.element_size(),
          t.size(1) == 1 ? t.size(2) : t.stride(1), t.size(0) == 1 ? 0 : t.stride(0)};
}

struct Heads {
  int64_t B, T, H, dk, dv;
};

bool width_ok(int64_t d) { return d == 32 || d == 64 || d == 128; }

Heads heads_of(const char* what, const Tensor& q, const Tensor& k, const Tensor& v, int64_t H, const Tensor& log_decay, int64_t dims) {
  TORCH_CHECK(known(q.scalar_type()) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), what, ": dtypes ",
              q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type(), "; supported: all float32 or all bfloat16");
  TORCH_CHECK(q.dim() == dims && k.sizes() == q.sizes() && v.dim() == dims && v.sizes().slice(0, dims - 1) == q.sizes().slice(0, dims - 1),
              what, ": q and k must share one ", dims == 3 ? "[batch, frames, channels]" : "[batch, channels]",
              " shape and v its leading dimensions, got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  on_gpu(what, "q", q, q, "q");
  on_gpu(what, "k", k, q, "q");
  on_gpu(what, "v", v, q, "q");
  on_gpu(what, "log_decay", log_decay, q, "q");
  const int64_t c = q.size(dims - 1), cv = v.size(dims - 1);
  TORCH_CHECK(H > 0 && c % H == 0 && cv % H == 0, what, ": ", c, " and ", cv, " channels do not split into ", H, " heads");
  TORCH_CHECK(width_ok(c / H) && width_ok(cv / H), what, ": head widths ", c / H, ", ", cv / H, "; supported: 32, 64, 128");
  TORCH_CHECK(log_decay.scalar_type() == at::kFloat && log_decay.dim() == 1 && log_decay.size(0) == H, what, ": log_decay must be float32 [",
              H, "], got ", log_decay.scalar_type(), " ", log_decay.sizes());
  TORCH_CHECK(!(log_decay.requires_grad() && at::GradMode::is_enabled()), what,
              ": the decays are constants; log_decay must not require a gradient");
  const int64_t T = dims == 3 ? q.size(1) : 1;
  TORCH_CHECK(q.size(0) <= INT32_MAX && T <= INT32_MAX && H <= INT32_MAX, what, ": too large, got ", q.sizes());
  return {q.size(0), T, H, c / H, cv / H};
}

void check_state(const char* what, const Tensor& state, const Tensor& q, const Heads& s) {
  TORCH_CHECK(state.scalar_type() == at::kFloat && state.sizes() == at::IntArrayRef({s.B, s.H, s.dk, s.dv}) && state.is_contiguous() &&
                  state.device() == q.device() && reinterpret_cast<uintptr_t>(state.const_data_ptr()) % 16 == 0,
              what, ": `state` must be a contiguous float32 tensor [", s.B, ", ", s.H, ", ", s.dk, ", ", s.dv, "] on ", q.device(),
              " that starts on a 16-byte boundary, got ", state.scalar_type(), " ", state.sizes(), " on ", state.device());
  TORCH_CHECK(!state.requires_grad(), what, ": `state` is replaced in place and must not require a gradient");
}

float scale_of(const std::optional<double>& scale, int64_t dk) { return (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)dk)); }

Tensor decay_run(const Rows& q, const Rows& k, const Rows& v, const Tensor& like, const Heads& s, const Tensor& log_decay,
                 const Tensor& lengths, const Tensor& state, float scale) {
  Tensor out = at::empty({s.B, s.T, s.H * s.dv}, like.options().requires_grad(false));
  const int dt = dtype_of(like);
  const size_t bytes = lib.lmufft_decay_workspace_bytes(dt, s.B, s.T, s.H, s.dk, s.dv, 0);
  Tensor ws = workspace(bytes, like);
  OnDevice on(like);
  ran(lib.lmufft_decay_attention(q.p, k.p, v.p, dt, q.ld, q.bs, k.ld, k.bs, v.ld, v.bs, log_decay.const_data_ptr<float>(),
                                 static_cast<const int32_t*>(ptr(lengths)), s.B, s.T, s.H, s.dk, s.dv, scale, out.mutable_data_ptr(),
                                 s.H * s.dv, s.T * s.H * s.dv, ptr_mut<float>(state), ptr_mut<void>(ws), bytes, on.stream),
      "lmufft_decay_attention");
  return out;
}

void decay_run_bwd(const Rows& q, const Rows& k, const Rows& v, const Tensor& like, Tensor dout, const Heads& s, const Tensor& log_decay,
                   const Tensor& lengths, float scale, const Rows& dq, const Rows& dk, const Rows& dv) {
  if (dout.scalar_type() != like.scalar_type()) dout = dout.to(like.scalar_type());
  dout = with_rows(dout);
  const Rows d = rows_of(dout);
  const int dt = dtype_of(like);
  const size_t bytes = lib.lmufft_decay_workspace_bytes(dt, s.B, s.T, s.H, s.dk, s.dv, 1);
  Tensor ws = workspace(bytes, like);
  OnDevice on(like);
  auto grad = [](const Rows& r) { return const_cast<void*>(r.p); };
  auto bs = [&](const Rows& r) { return s.B == 1 ? s.T * r.ld : r.bs; };
  ran(lib.lmufft_decay_attention_bwd(q.p, k.p, v.p, d.p, dt, q.ld, q.bs, k.ld, k.bs, v.ld, v.bs, d.ld, d.bs,
                                     log_decay.const_data_ptr<float>(), static_cast<const int32_t*>(ptr(lengths)), s.B, s.T, s.H, s.dk,
                                     s.dv, scale, grad(dq), grad(dk), grad(dv), dq.ld, bs(dq), dk.ld, bs(dk), dv.ld, bs(dv),
                                     ptr_mut<void>(ws), bytes, on.stream),
      "lmufft_decay_attention_bwd");
}

Tensor decay_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t num_heads, const Tensor& log_decay,
                       const MaybeTensor& lengths, const MaybeTensor& state, std::optional<double> scale) {
  const char* what = "decay_attention";
  const Heads s = heads_of(what, q, k, v, num_heads, log_decay, 3);
  if (state) check_state(what, *state, q, s);
  const Tensor n = frames_of(what, "lengths", lengths, q, s.B);
  at::NoGradGuard no_grad;
  const Tensor qr = with_rows(q), kr = with_rows(k), vr = with_rows(v);
  Tensor out = decay_run(rows_of(qr), rows_of(kr), rows_of(vr), q, s, log_decay.contiguous(), n, state.value_or(Tensor()),
                         scale_of(scale, s.dk));
  if (state) torch::autograd::impl::bump_version(*state);
  return out;
}

Tensor decay_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, int64_t num_heads, const Tensor& log_decay,
                            const Tensor& state, const MaybeTensor& active, std::optional<double> scale) {
  const char* what = "decay_attention_step";
  const Heads s = heads_of(what, q, k, v, num_heads, log_decay, 2);
  check_state(what, state, q, s);
  const Tensor n = frames_of(what, "active", active, q, s.B);
  at::NoGradGuard no_grad;
  auto row = [](const Tensor& t) { return t.stride(1) == 1 ? t : t.contiguous(); };
  const Tensor qr = row(q), kr = row(k), vr = row(v), ld = log_decay.contiguous();
  Tensor out = at::empty({s.B, s.H * s.dv}, q.options().requires_grad(false));
  OnDevice on(q);
  ran(lib.lmufft_decay_attention_step(qr.const_data_ptr(), kr.const_data_ptr(), vr.const_data_ptr(), dtype_of(q), qr.stride(0),
                                      kr.stride(0), vr.stride(0), ld.const_data_ptr<float>(), static_cast<const int32_t*>(ptr(n)), s.B,
                                      s.H, s.dk, s.dv, scale_of(scale, s.dk), out.mutable_data_ptr(), s.H * s.dv,
                                      static_cast<float*>(state.mutable_data_ptr()), on.stream),
      "lmufft_decay_attention_step");
  torch::autograd::impl::bump_version(state);
  return out;
}

// What a training call carries besides its differentiable tensors.
struct DecayCall {
  Tensor log_decay, lengths;
  int64_t H;
  double scale;
};

struct DecayTrain : torch::autograd::Function<DecayTrain> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const DecayCall& a) {
    const Tensor q = with_rows(q_), k = with_rows(k_), v = with_rows(v_);
    const int64_t H = a.H;
    const Heads s{q.size(0), q.size(1), H, q.size(2) / H, v.size(2) / H};
    ctx->save_for_backward({q, k, v, a.log_decay, a.lengths});
    ctx->saved_data["heads"] = H;
    ctx->saved_data["scale"] = a.scale;
    return decay_run(rows_of(q), rows_of(k), rows_of(v), q, s, a.log_decay, a.lengths, Tensor(), (float)a.scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2];
    const int64_t H = ctx->saved_data["heads"].toInt();
    const Heads s{q.size(0), q.size(1), H, q.size(2) / H, v.size(2) / H};
    variable_list out(4);
    {
      at::NoGradGuard no_grad;
      const auto options = q.options().requires_grad(false);
      out[0] = at::empty(q.sizes(), options), out[1] = at::empty(k.sizes(), options), out[2] = at::empty(v.sizes(), options);
      decay_run_bwd(rows_of(q), rows_of(k), rows_of(v), q, grads[0], s, saved[3], saved[4], (float)ctx->saved_data["scale"].toDouble(),
                    rows_of(out[0]), rows_of(out[1]), rows_of(out[2]));
    }
    return once("decay_attention_train", std::move(out));
  }
};

struct DecayTrainPacked : torch::autograd::Function<DecayTrainPacked> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv_, const DecayCall& a) {
    const Tensor qkv = with_rows(qkv_);
    const int64_t H = a.H, c = qkv.size(2) / 3;
    ctx->save_for_backward({qkv, a.log_decay, a.lengths});
    ctx->saved_data["heads"] = H;
    ctx->saved_data["scale"] = a.scale;
    return decay_run(rows_of(qkv), rows_of(qkv, c), rows_of(qkv, 2 * c), qkv, Heads{qkv.size(0), qkv.size(1), H, c / H, c / H},
                     a.log_decay, a.lengths, Tensor(), (float)a.scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& qkv = saved[0];
    const int64_t H = ctx->saved_data["heads"].toInt(), c = qkv.size(2) / 3;
    variable_list out(2);
    {
      at::NoGradGuard no_grad;
      Tensor g = at::empty(qkv.sizes(), qkv.options().requires_grad(false));
      decay_run_bwd(rows_of(qkv), rows_of(qkv, c), rows_of(qkv, 2 * c), qkv, grads[0],
                    Heads{qkv.size(0), qkv.size(1), H, c / H, c / H}, saved[1], saved[2], (float)ctx->saved_data["scale"].toDouble(),
                    rows_of(g), rows_of(g, c), rows_of(g, 2 * c));
      out[0] = g;
    }
    return once("decay_attention_train_packed", std::move(out));
  }
};

Tensor decay_attention_train(const Tensor& q, const Tensor& k, const Tensor& v, int64_t num_heads, const Tensor& log_decay,
                             const MaybeTensor& lengths, std::optional<double> scale) {
  const char* what = "decay_attention_train";
  const Heads s = heads_of(what, q, k, v, num_heads, log_decay, 3);
  return DecayTrain::apply(q, k, v, DecayCall{log_decay.contiguous(), frames_of(what, "lengths", lengths, q, s.B), num_heads,
                                              (double)scale_of(scale, s.dk)});
}

Tensor decay_attention_train_packed(const Tensor& qkv, int64_t num_heads, const Tensor& log_decay, const MaybeTensor& lengths,
                                    std::optional<double> scale) {
  const char* what = "decay_attention_train_packed";
  TORCH_CHECK(qkv.dim() == 3 && qkv.size(2) % 3 == 0, what, ": qkv must be [batch, frames, 3 * channels], got ", qkv.sizes());
  Heads s;
  {
    at::NoGradGuard no_grad;
    const Tensor q = qkv.narrow(2, 0, qkv.size(2) / 3);
    s = heads_of(what, q, q, q, num_heads, log_decay, 3);
  }
  TORCH_CHECK(!(log_decay.requires_grad() && at::GradMode::is_enabled()), what,
              ": the decays are constants; log_decay must not require a gradient");
  return DecayTrainPacked::apply(qkv, DecayCall{log_decay.contiguous(), frames_of(what, "lengths", lengths, qkv, s.B), num_heads,
                                                (double)scale_of(scale, s.dk)});
}

// ---- group norm (asr_amd/groupnorm.py)
constexpr int64_t kGroupNormMaxWidth = 1024;

struct Sample {
  int64_t N, T, C;
};
Sample sample_of(const Tensor& x) { return x.dim() == 2 ? Sample{x.size(0), 1, x.size(1)} : Sample{x.size(0), x.size(1), x.size(2)}; }

struct NormArgs {
  int64_t groups;
  double eps;
  int act;
  at::ScalarType out;
  Tensor lengths;
};

NormArgs norm_args(const char* what, const Tensor& x, int64_t groups, const Tensor& weight, const Tensor& bias, double eps,
                   const std::optional<std::string>& activation, const MaybeTensor& lengths, const std::optional<at::ScalarType>& out_dtype) {
  const at::ScalarType out = out_dtype ? *out_dtype : at::autocast::is_autocast_enabled(at::kCUDA) ? at::kFloat : x.scalar_type();
  TORCH_CHECK(known(x.scalar_type()) && known(out), what, ": supported dtypes are float32 and bfloat16, got ", x.scalar_type(),
              " and an output of ", out);
  TORCH_CHECK(x.dim() == 2 || x.dim() == 3, what, ": x must be [batch, frames, channels] or [rows, channels], got ", x.sizes());
  const int64_t C = x.size(-1);
  TORCH_CHECK(groups > 0 && C > 0 && C % groups == 0, what, ": ", C, " channels do not split into ", groups, " groups");
  TORCH_CHECK(C <= kGroupNormMaxWidth, what, ": ", C, " channels; at most ", kGroupNormMaxWidth);
  int act = -1;
  if (!activation) act = 0;
  else if (*activation == "relu") act = 1;
  else if (*activation == "silu") act = 2;
  TORCH_CHECK(act >= 0, what, ": activation '", *activation, "'; supported: None, 'relu', 'silu'");
  on_gpu(what, "x", x, x, "x");
  on_gpu(what, "weight", weight, x, "x");
  on_gpu(what, "bias", bias, x, "x");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == C && bias.dim() == 1 && bias.size(0) == C, what,
              ": weight and bias must have shape (", C, ",)");
  TORCH_CHECK(x.dim() == 3 || !lengths.has_value(), what, ": lengths go with x of shape [batch, frames, channels]");
  TORCH_CHECK(x.size(0) <= INT64_MAX / 2048 && (x.dim() == 2 || x.size(1) <= INT32_MAX), what, ": too large, got ", x.sizes());
  return {groups, eps, act, out, x.dim() == 3 ? frames_of(what, "lengths", lengths, x, x.size(0)) : Tensor()};
}

// x, weight, bias dense; weight, bias float32
Tensor norm_run(const Tensor& x, const Tensor& weight, const Tensor& bias, const NormArgs& a, bool with_stats, Tensor* stats) {
  const Sample s = sample_of(x);
  Tensor out = at::empty(x.sizes(), x.options().dtype(a.out).requires_grad(false));
  if (with_stats && (s.T > 1 || a.lengths.defined()))
    *stats = at::empty({s.N, a.groups, 2}, x.options().dtype(at::kDouble).requires_grad(false));
  const size_t bytes = lib.lmufft_group_norm_workspace_bytes(s.N, s.T, s.C, a.groups, 0);
  Tensor ws = workspace(bytes, x);
  OnDevice on(x);
  ran(lib.lmufft_group_norm(x.const_data_ptr(), dtype_of(x), weight.const_data_ptr<float>(), bias.const_data_ptr<float>(),
                            static_cast<const int32_t*>(ptr(a.lengths)), s.N, s.T, s.C, a.groups, (float)a.eps, a.act,
                            out.mutable_data_ptr(), dtype_of(out), with_stats ? ptr_mut<double>(*stats) : nullptr, ptr_mut<void>(ws), bytes,
                            on.stream),
      "lmufft_group_norm");
  return out;
}

Tensor as_param(const Tensor& t) { return dense(t.scalar_type() == at::kFloat ? t : t.to(at::kFloat)); }

Tensor group_norm(const Tensor& x, int64_t num_groups, const Tensor& weight, const Tensor& bias, double eps,
                  const std::optional<std::string>& activation, const MaybeTensor& lengths, const std::optional<at::ScalarType>& out_dtype) {
  const NormArgs a = norm_args("group_norm", x, num_groups, weight, bias, eps, activation, lengths, out_dtype);
  at::NoGradGuard no_grad;
  return norm_run(dense(x), as_param(weight), as_param(bias), a, false, nullptr);
}

struct GroupNormTrain : torch::autograd::Function<GroupNormTrain> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& weight, const Tensor& bias, const NormArgs& a) {
    const Tensor x = dense(x_), w = as_param(weight), b = as_param(bias);
    Tensor stats;
    Tensor out = norm_run(x, w, b, a, true, &stats);
    ctx->save_for_backward({x, w, b, a.lengths, stats});
    ctx->saved_data["groups"] = a.groups;
    ctx->saved_data["eps"] = a.eps;
    ctx->saved_data["act"] = (int64_t)a.act;
    ctx->saved_data["weight"] = (int64_t)weight.scalar_type();
    ctx->saved_data["bias"] = (int64_t)bias.scalar_type();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &lengths = saved[3], &stats = saved[4];
    const int64_t groups = ctx->saved_data["groups"].toInt();
    const Sample s = sample_of(x);
    variable_list out(4);
    {
      at::NoGradGuard no_grad;
      const Tensor dy = dense(known(grads[0].scalar_type()) ? grads[0] : grads[0].to(at::kFloat));
      out[0] = at::empty(x.sizes(), x.options().requires_grad(false));
      const auto f32 = x.options().dtype(at::kFloat).requires_grad(false);
      out[1] = at::empty({s.C}, f32), out[2] = at::empty({s.C}, f32);
      const size_t bytes = lib.lmufft_group_norm_workspace_bytes(s.N, s.T, s.C, groups, 1);
      Tensor ws = workspace(bytes, x);
      OnDevice on(x);
      ran(lib.lmufft_group_norm_bwd(x.const_data_ptr(), dtype_of(x), dy.const_data_ptr(), dtype_of(dy), w.const_data_ptr<float>(),
                                    b.const_data_ptr<float>(), static_cast<const int32_t*>(ptr(lengths)),
                                    static_cast<const double*>(ptr(stats)), s.N, s.T, s.C, groups, (float)ctx->saved_data["eps"].toDouble(),
                                    (int)ctx->saved_data["act"].toInt(), out[0].mutable_data_ptr(), out[1].mutable_data_ptr<float>(),
                                    out[2].mutable_data_ptr<float>(), ptr_mut<void>(ws), bytes, on.stream),
          "lmufft_group_norm_bwd");
      const auto wt = (at::ScalarType)ctx->saved_data["weight"].toInt(), bt = (at::ScalarType)ctx->saved_data["bias"].toInt();
      if (wt != at::kFloat) out[1] = out[1].to(wt);
      if (bt != at::kFloat) out[2] = out[2].to(bt);
    }
    return once("group_norm_train", std::move(out));
  }
};

Tensor group_norm_train(const Tensor& x, int64_t num_groups, const Tensor& weight, const Tensor& bias, double eps,
                        const std::optional<std::string>& activation, const MaybeTensor& lengths,
                        const std::optional<at::ScalarType>& out_dtype) {
  return GroupNormTrain::apply(x, weight, bias, norm_args("group_norm_train", x, num_groups, weight, bias, eps, activation, lengths, out_dtype));
}

// ---- residual dropout (asr_amd/dropout.py)
Tensor dropout_run(const Tensor& x, const Tensor& residual, double p, int64_t seed0, int64_t seed1, at::ScalarType out_dtype) {
  Tensor out = at::empty(x.sizes(), x.options().dtype(out_dtype).requires_grad(false));
  const int64_t C = x.size(-1);
  OnDevice on(x);
  ran(lib.lmufft_dropout_add(x.const_data_ptr(), dtype_of(x), ptr(residual), residual.defined() ? dtype_of(residual) : 0, x.numel() / C, C,
                             (float)p, (uint32_t)seed0, (uint32_t)seed1, out.mutable_data_ptr(), dtype_of(out), on.stream),
      "lmufft_dropout_add");
  return out;
}

struct DropoutAdd : torch::autograd::Function<DropoutAdd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual, double p, int64_t seed0, int64_t seed1,
                        at::ScalarType out_dtype) {
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed0"] = seed0;
    ctx->saved_data["seed1"] = seed1;
    ctx->saved_data["x"] = (int64_t)x.scalar_type();
    ctx->saved_data["added"] = residual.has_value();
    ctx->saved_data["residual"] = (int64_t)(residual ? *residual : x).scalar_type();
    return dropout_run(dense(x), residual ? dense(*residual) : Tensor(), p, seed0, seed1, out_dtype);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    {
      at::NoGradGuard no_grad;
      const Tensor dy = known(grads[0].scalar_type()) ? grads[0] : grads[0].to(at::kFloat);
      if (ctx->needs_input_grad(0))
        out[0] = dropout_run(dense(dy), Tensor(), ctx->saved_data["p"].toDouble(), ctx->saved_data["seed0"].toInt(),
                             ctx->saved_data["seed1"].toInt(), (at::ScalarType)ctx->saved_data["x"].toInt());
      if (ctx->saved_data["added"].toBool() && ctx->needs_input_grad(1)) out[1] = grads[0].to((at::ScalarType)ctx->saved_data["residual"].toInt());
    }
    return once("dropout_add", std::move(out));
  }
};

Tensor dropout_add(const Tensor& x, const MaybeTensor& residual, double p, int64_t seed0, int64_t seed1,
                   const std::optional<at::ScalarType>& out_dtype) {
  const char* what = "dropout_add";
  auto fit = [&](const char* name, const Tensor& t) {
    TORCH_CHECK(known(t.scalar_type()), what, ": `", name, "` is ", t.scalar_type(), "; supported dtypes are float32 and bfloat16");
    on_gpu(what, name, t, x, "x");
  };
  fit("x", x);
  if (residual) fit("residual", *residual);
  TORCH_CHECK(x.dim() > 0 && x.size(-1) > 0 && x.size(-1) <= INT32_MAX, what, ": x must be [..., channels], got ", x.sizes());
  TORCH_CHECK(!residual || residual->sizes() == x.sizes(), what, ": residual does not match x, got ", x.sizes());
  const at::ScalarType out = out_dtype ? *out_dtype : residual ? at::promote_types(x.scalar_type(), residual->scalar_type()) : x.scalar_type();
  TORCH_CHECK(known(out), what, ": output dtype ", out, " is not supported");
  return DropoutAdd::apply(x, residual, p, seed0, seed1, out);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  typedef py::call_guard<py::gil_scoped_release> free_gil;
  m.def("bind", &bind);
  m.def("decay_attention", &decay_attention, free_gil());
  m.def("decay_attention_step", &decay_attention_step, free_gil());
  m.def("decay_attention_train", &decay_attention_train, free_gil());
  m.def("decay_attention_train_packed", &decay_attention_train_packed, free_gil());
  m.def("group_norm", &group_norm, free_gil());
  m.def("group_norm_train", &group_norm_train, free_gil());
  m.def("dropout_add", &dropout_add, free_gil());
  m.attr("abi_version") = LMUFFT_ABI_VERSION;  // of the signatures compiled in
  m.attr("entries") = py::make_tuple(
#define X(name) #name,
      LMUFFT_ENTRIES(X)
#undef X
          "");
}
