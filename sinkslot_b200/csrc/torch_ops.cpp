// torch_ops.cpp -- the training operators as PyTorch operators
// (torch.ops.sinkslot_b200.*) with their argument checks and their autograd, over
// the C entries of libsinkslot_b200.so.
//
// They are called on small tensors many times a step, where the host's own time
// is the call's: a forward and backward pass through Python autograd functions
// and a ctypes binding took 135 to 160 us, of which the kernels ran 3 to 10.
//
// Two layers: operators that launch (CUDA only; PyTorch sees their inputs and
// outputs), and the functions users call, which check, record the gradient and
// call the former (any dispatch mode, fake tensors among them).
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>

#include "../../include/sinkslot_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// ---------------------------------------------------------------------------
// Calls of the C entries
// ---------------------------------------------------------------------------
void done(int status, const char* name) {
  if (status == 0) return;
  TORCH_CHECK_VALUE(status != 1, name, ": ", sinkslot_last_error());
  TORCH_CHECK(false, name, " failed (status ", status, "): ", sinkslot_last_error());
}

int dtype_code(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kHalf ? 1 : 2;
}
void* ptr(const Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }
template <typename T>
T* ptr(const optional<Tensor>& t) {
  return t.has_value() && t->defined() && t->numel() ? static_cast<T*>(t->data_ptr()) : nullptr;
}
float* f32(const Tensor& t) { return static_cast<float*>(ptr(t)); }
void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}
Tensor empty_f32(at::IntArrayRef shape, const Tensor& like) {
  return at::empty(shape, like.options().dtype(at::kFloat));
}
Tensor workspace(int64_t bytes, const Tensor& like) {
  return at::empty({bytes}, like.options().dtype(at::kByte));
}

// An uninitialised (rows, vocab) tensor for the gradient of z: rows beginning on the
// same 16-byte phases as those of z (then both are read and written in whole vectors),
// contiguous where the rows of z overlap.  Rows of a padded buffer are as far apart as
// there; rows of a wider view (the last position of each sequence, every eighth row)
// only as far as the phase asks: their own distance would be memory of the buffer's size.
Tensor grad_like(const Tensor& z) {
  const int64_t rows = z.size(0), vocab = z.size(1), lanes = 16 / z.element_size();
  int64_t stride = z.stride(0);
  if (stride < vocab || rows <= 1)
    stride = vocab;
  else if (stride - vocab > std::max<int64_t>(vocab / 8, 256))
    stride = vocab + (stride - vocab) % lanes;
  const int64_t phase =
      rows ? (int64_t)(reinterpret_cast<uintptr_t>(z.const_data_ptr()) % 16) / z.element_size() : 0;
  if (stride == vocab && phase == 0) return at::empty({rows, vocab}, z.options());
  Tensor flat = at::empty({phase + (rows - 1) * stride + vocab}, z.options());
  return flat.as_strided({rows, vocab}, {stride, 1}, phase);
}

int64_t sequences(const optional<Tensor>& offsets) {
  return offsets.has_value() ? offsets->numel() - 1 : 1;
}
int offset_bytes(const optional<Tensor>& offsets) {
  return offsets.has_value() ? (int)offsets->element_size() : 8;
}

// What a launching operator takes for granted of its tensors (the functions above
// them see to it; a direct call that does not is refused).
void expect(const Tensor& t, at::ScalarType type, int64_t numel, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.scalar_type() == type && t.numel() == numel &&
                        t.is_contiguous(),
                    what, ": expected a contiguous CUDA tensor of ", numel, " ", type, ", got ",
                    t.sizes(), " ", t.scalar_type());
}
void expect(const optional<Tensor>& t, at::ScalarType type, int64_t numel, const char* what) {
  if (t.has_value()) expect(*t, type, numel, what);
}
void expect_index(const Tensor& t, int64_t numel, const char* what) {
  expect(t, t.scalar_type() == at::kInt ? at::kInt : at::kLong, numel, what);
}
void expect_rows(const Tensor& t, const char* what) {
  const auto d = t.scalar_type();
  TORCH_CHECK_VALUE(t.is_cuda() && t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1) &&
                        (d == at::kFloat || d == at::kHalf || d == at::kBFloat16),
                    what, ": expected rows of contiguous float32, float16 or bfloat16, got ",
                    t.sizes(), " ", d);
}
void expect_offsets(const optional<Tensor>& offsets) {
  if (!offsets.has_value()) return;
  TORCH_CHECK_VALUE(offsets->numel() >= 2, "offsets: expected two values or more");
  expect_index(*offsets, offsets->numel(), "offsets");
}

// ---------------------------------------------------------------------------
// Operators that launch
// ---------------------------------------------------------------------------
Tensor lookup(const Tensor& table, const Tensor& index, double scale) {
  expect_rows(table, "table");
  expect_index(index, index.numel(), "index");
  const c10::cuda::CUDAGuard guard(table.device());
  Tensor out = at::empty({index.numel(), table.size(1)}, table.options());
  done(sinkslot_lookup(ptr(table), dtype_code(table), table.stride(0), table.size(0),
                       table.size(1), ptr(index), (int)index.element_size(), index.numel(), scale,
                       ptr(out), stream_of(table)),
       "lookup");
  return out;
}

Tensor lookup_grad(const Tensor& grad_out, const Tensor& index, int64_t rows, double scale,
                   int64_t padding) {
  const c10::cuda::CUDAGuard guard(grad_out.device());
  TORCH_CHECK_VALUE(grad_out.dim() == 2 && grad_out.size(0) == index.numel(),
                    "grad_out: expected a row for each index");
  expect_index(index, index.numel(), "index");
  const Tensor g = grad_out.stride(1) == 1 || grad_out.size(1) == 1 ? grad_out
                                                                     : grad_out.contiguous();
  expect_rows(g, "grad_out");
  const int64_t dim = g.size(1), count = index.numel();
  int64_t bytes = 0;
  done(sinkslot_lookup_grad_workspace_bytes(count, rows, dim, &bytes), "lookup_grad");
  Tensor ws = workspace(bytes, g);
  Tensor out = at::empty({rows, dim}, g.options());
  done(sinkslot_lookup_grad(ptr(g), dtype_code(g), g.stride(0), ptr(index),
                            (int)index.element_size(), count, rows, dim, scale, padding, ptr(out),
                            ptr(ws), bytes, stream_of(g)),
       "lookup_grad");
  return out;
}

std::tuple<Tensor, Tensor, Tensor> token_logprobs(const Tensor& z, const Tensor& tokens,
                                                  double temperature, int64_t ignore_index,
                                                  bool entropy) {
  expect_rows(z, "logits");
  expect_index(tokens, z.size(0), "tokens");
  const c10::cuda::CUDAGuard guard(z.device());
  const int64_t rows = z.size(0);
  Tensor logp = empty_f32({rows}, z), ent = empty_f32({entropy ? rows : 0}, z),
         stats = empty_f32({rows, 2}, z);
  done(sinkslot_token_logprobs(ptr(z), dtype_code(z), z.stride(0), rows, z.size(1), ptr(tokens),
                               (int)tokens.element_size(), ignore_index, 1.0 / temperature,
                               f32(logp), f32(ent), f32(stats), stream_of(z)),
       "token_logprobs");
  return {logp, ent, stats};
}

Tensor token_logprobs_grad(const Tensor& z, const Tensor& tokens, const Tensor& stats,
                           const Tensor& entropy, const optional<Tensor>& g,
                           const optional<Tensor>& g_entropy, double temperature,
                           int64_t ignore_index) {
  expect_rows(z, "logits");
  const int64_t rows = z.size(0);
  expect_index(tokens, rows, "tokens");
  expect(stats, at::kFloat, 2 * rows, "stats");
  expect(entropy, at::kFloat, g_entropy.has_value() ? rows : entropy.numel(), "entropy");
  for (const auto* t : {&g, &g_entropy})  // one value may stand for all rows
    TORCH_CHECK_VALUE(!t->has_value() || ((*t)->is_cuda() && (*t)->scalar_type() == at::kFloat &&
                                          (*t)->dim() == 1 && (*t)->numel() == rows),
                      "outer gradient: expected one float32 for each row");
  const c10::cuda::CUDAGuard guard(z.device());
  Tensor out = grad_like(z);
  done(sinkslot_token_logprobs_grad(
           ptr(z), dtype_code(z), z.stride(0), z.size(0), z.size(1), ptr(tokens),
           (int)tokens.element_size(), ignore_index, 1.0 / temperature, f32(stats), f32(entropy),
           ptr<float>(g), g.has_value() ? g->stride(0) : 0, ptr<float>(g_entropy),
           g_entropy.has_value() ? g_entropy->stride(0) : 0, ptr(out), out.stride(0),
           stream_of(z)),
       "token_logprobs_grad");
  return out;
}

std::tuple<Tensor, Tensor> policy_loss(const Tensor& logp, const Tensor& old_logp,
                                       const Tensor& advantages, const optional<Tensor>& ref_logp,
                                       const optional<Tensor>& mask,
                                       const optional<Tensor>& offsets, bool adv_per_token,
                                       double clip_low, double clip_high, double kl_coef,
                                       int64_t kl, bool sequence_average, bool want_grad) {
  expect_offsets(offsets);
  const int64_t t = logp.numel(), s = sequences(offsets);
  expect(logp, at::kFloat, t, "logp");
  expect(old_logp, at::kFloat, t, "old_logp");
  expect(ref_logp, at::kFloat, t, "ref_logp");
  expect(advantages, at::kFloat, adv_per_token ? t : s, "advantages");
  expect(mask, at::kBool, t, "mask");
  const c10::cuda::CUDAGuard guard(logp.device());
  int64_t bytes = 0;
  done(sinkslot_loss_workspace_bytes(s, &bytes), "policy_loss");
  Tensor ws = workspace(bytes, logp), values = empty_f32({4}, logp),
         coef = empty_f32({want_grad ? t : 0}, logp);
  done(sinkslot_policy_loss(f32(logp), f32(old_logp), ptr<float>(ref_logp), f32(advantages),
                            adv_per_token, ptr<uint8_t>(mask), ptr<void>(offsets),
                            offset_bytes(offsets), s, t, clip_low, clip_high, kl_coef, (int)kl,
                            sequence_average, f32(values), f32(coef), ptr(ws), bytes,
                            stream_of(logp)),
       "policy_loss");
  return {values, coef};
}

Tensor scale_tokens(const Tensor& coef, const Tensor& values, const Tensor& g) {
  expect(coef, at::kFloat, coef.numel(), "coef");
  expect(values, at::kFloat, 4, "values");
  expect(g, at::kFloat, 1, "outer gradient");
  const c10::cuda::CUDAGuard guard(coef.device());
  Tensor out = at::empty_like(coef);
  done(sinkslot_scale_tokens(f32(coef), coef.numel(), f32(values) + 3, f32(g), f32(out),
                             stream_of(coef)),
       "scale_tokens");
  return out;
}

std::tuple<Tensor, Tensor, Tensor> policy_loss_logits(
    const Tensor& z, const Tensor& tokens, const Tensor& old_logp, const Tensor& advantages,
    const optional<Tensor>& ref_logp, const optional<Tensor>& mask,
    const optional<Tensor>& offsets, double temperature, bool adv_per_token, double clip_low,
    double clip_high, double kl_coef, int64_t kl, bool sequence_average, double grad_scale,
    bool want_grad) {
  expect_rows(z, "logits");
  expect_offsets(offsets);
  const int64_t t = z.size(0), vocab = z.size(1), s = sequences(offsets);
  expect_index(tokens, t, "tokens");
  expect(old_logp, at::kFloat, t, "old_logp");
  expect(ref_logp, at::kFloat, t, "ref_logp");
  expect(advantages, at::kFloat, adv_per_token ? t : s, "advantages");
  expect(mask, at::kBool, t, "mask");
  const c10::cuda::CUDAGuard guard(z.device());
  int64_t bytes = 0;
  done(sinkslot_policy_logits_workspace_bytes(t, s, &bytes), "policy_loss_from_logits");
  Tensor ws = workspace(bytes, z), values = empty_f32({4}, z), logp = empty_f32({t}, z);
  Tensor grad = want_grad ? grad_like(z) : at::empty({0, vocab}, z.options());
  done(sinkslot_policy_loss_logits(
           ptr(z), dtype_code(z), z.stride(0), t, vocab, ptr(tokens), (int)tokens.element_size(),
           1.0 / temperature, f32(old_logp), ptr<float>(ref_logp), f32(advantages), adv_per_token,
           ptr<uint8_t>(mask), ptr<void>(offsets), offset_bytes(offsets), s, clip_low, clip_high,
           kl_coef, (int)kl, sequence_average, grad_scale, f32(values), f32(logp), ptr(grad),
           grad.stride(0), ptr(ws), bytes, stream_of(z)),
       "policy_loss_from_logits");
  return {values, logp, grad};
}

void scale_rows_(Tensor grad, const Tensor& g, double grad_scale) {
  expect_rows(grad, "grad");
  expect(g, at::kFloat, 1, "outer gradient");
  const c10::cuda::CUDAGuard guard(grad.device());
  done(sinkslot_scale_rows(ptr(grad), dtype_code(grad), grad.stride(0), grad.size(0),
                           grad.size(1), f32(g), grad_scale, stream_of(grad)),
       "scale_rows");
}

std::tuple<Tensor, Tensor, Tensor> preference_loss(const Tensor& logp, const Tensor& offsets,
                                                   const optional<Tensor>& ref_logp,
                                                   const optional<Tensor>& mask, double beta,
                                                   double smoothing, int64_t kind,
                                                   bool normalize) {
  expect_offsets(offsets);
  expect(logp, at::kFloat, logp.numel(), "logp");
  expect(ref_logp, at::kFloat, logp.numel(), "ref_logp");
  expect(mask, at::kBool, logp.numel(), "mask");
  const c10::cuda::CUDAGuard guard(logp.device());
  const int64_t s = offsets.numel() - 1;
  int64_t bytes = 0;
  done(sinkslot_loss_workspace_bytes(s, &bytes), "preference_loss");
  Tensor ws = workspace(bytes, logp), loss = empty_f32({}, logp), rewards = empty_f32({s}, logp),
         slope = empty_f32({s}, logp);
  done(sinkslot_preference_loss(f32(logp), ptr<float>(ref_logp), ptr<uint8_t>(mask), ptr(offsets),
                                (int)offsets.element_size(), s, logp.numel(), beta, smoothing,
                                (int)kind, normalize, f32(loss), f32(rewards), f32(slope), ptr(ws),
                                bytes, stream_of(logp)),
       "preference_loss");
  return {loss, rewards, slope};
}

Tensor preference_grad(const Tensor& slope, const Tensor& offsets, const optional<Tensor>& mask,
                       const Tensor& g, int64_t tokens) {
  expect(slope, at::kFloat, slope.numel(), "slope");
  expect_index(offsets, slope.numel() + 1, "offsets");
  expect(mask, at::kBool, tokens, "mask");
  expect(g, at::kFloat, 1, "outer gradient");
  const c10::cuda::CUDAGuard guard(slope.device());
  Tensor out = empty_f32({tokens}, slope);
  done(sinkslot_preference_grad(f32(slope), ptr<uint8_t>(mask), ptr(offsets),
                                (int)offsets.element_size(), slope.numel(), tokens, f32(g),
                                f32(out), stream_of(slope)),
       "preference_grad");
  return out;
}

// The launching operators, called through the dispatcher.

#define SINKSLOT_OP(fn)                                                             \
  c10::TypedOperatorHandle<decltype(fn)> fn##_op() {                                \
    static const auto handle = c10::Dispatcher::singleton()                         \
                                   .findSchemaOrThrow("sinkslot_b200::" #fn, "")    \
                                   .typed<decltype(fn)>();                          \
    return handle;                                                                  \
  }
SINKSLOT_OP(lookup)
SINKSLOT_OP(lookup_grad)
SINKSLOT_OP(token_logprobs)
SINKSLOT_OP(token_logprobs_grad)
SINKSLOT_OP(policy_loss)
SINKSLOT_OP(scale_tokens)
SINKSLOT_OP(policy_loss_logits)
SINKSLOT_OP(scale_rows_)
SINKSLOT_OP(preference_loss)
SINKSLOT_OP(preference_grad)

// ---------------------------------------------------------------------------
// Autograd
// ---------------------------------------------------------------------------

// A backward pass recorded for a second derivative: the gradient is handed out,
// and differentiating it again is an error.
template <typename F>
Tensor first_order(const char* name, F&& compute) {
  if (!at::GradMode::is_enabled()) return compute();
  Tensor out;
  {
    at::NoGradGuard off;
    out = compute();
  }
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("sinkslot_b200: ") + name + " has no second derivative", 1);
  out.set_requires_grad(true);
  return (*error)({out})[0];
}

variable_list first_of(int n, Tensor grad) {
  variable_list v((size_t)n);
  v[0] = std::move(grad);
  return v;
}

struct LookupFn : Function<LookupFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& index,
                        double scale, int64_t padding) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({index});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return lookup_op().call(table, index, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    return first_of(4, first_order("embedding_lookup", [&] {
      return lookup_grad_op().call(g[0], saved[0], ctx->saved_data["rows"].toInt(),
                                   ctx->saved_data["scale"].toDouble(),
                                   ctx->saved_data["padding"].toInt());
    }));
  }
};

struct TokenLogprobsFn : Function<TokenLogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& tokens,
                               double temperature, int64_t ignore_index, bool entropy) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->set_materialize_grads(false);
    auto [logp, ent, stats] =
        token_logprobs_op().call(z, tokens, temperature, ignore_index, entropy);
    ctx->save_for_backward({z, tokens, stats, ent});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore_index;
    if (entropy) return {logp, ent};
    return {logp};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const Tensor ge = g.size() > 1 ? g[1] : Tensor();
    if (!g[0].defined() && !ge.defined()) return variable_list(5);
    const auto s = ctx->get_saved_variables();
    auto maybe = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; };
    return first_of(5, first_order("token_logprobs", [&] {
      return token_logprobs_grad_op().call(s[0], s[1], s[2], s[3], maybe(g[0]), maybe(ge),
                                           ctx->saved_data["temperature"].toDouble(),
                                           ctx->saved_data["ignore"].toInt());
    }));
  }
};

// Options of the policy loss behind its tensors.
struct PolicyArgs {
  bool adv_per_token;
  double clip_low, clip_high, kl_coef;
  int64_t kl;
  bool sequence_average;
};

struct PolicyLossFn : Function<PolicyLossFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logp, const Tensor& old_logp,
                               const Tensor& adv, const optional<Tensor>& ref,
                               const optional<Tensor>& mask, const optional<Tensor>& offsets,
                               PolicyArgs a) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [values, coef] = policy_loss_op().call(logp, old_logp, adv, ref, mask, offsets,
                                                a.adv_per_token, a.clip_low, a.clip_high,
                                                a.kl_coef, a.kl, a.sequence_average, true);
    ctx->save_for_backward({values, coef});
    ctx->set_materialize_grads(false);
    auto v = values.unbind();
    ctx->mark_non_differentiable({v[1], v[2]});
    return {v[0], v[1], v[2]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return variable_list(7);
    const auto s = ctx->get_saved_variables();
    return first_of(7, first_order("policy_loss", [&] {
      return scale_tokens_op().call(s[1], s[0], g[0]);
    }));
  }
};

struct PolicyLossLogitsFn : Function<PolicyLossLogitsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& tokens,
                               const Tensor& old_logp, const Tensor& adv,
                               const optional<Tensor>& ref, const optional<Tensor>& mask,
                               const optional<Tensor>& offsets, double temperature, PolicyArgs a,
                               double grad_scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [values, logp, grad] = policy_loss_logits_op().call(
        z, tokens, old_logp, adv, ref, mask, offsets, temperature, a.adv_per_token, a.clip_low,
        a.clip_high, a.kl_coef, a.kl, a.sequence_average, grad_scale, true);
    ctx->saved_data["grad"] = grad;
    ctx->saved_data["scale"] = grad_scale;
    ctx->set_materialize_grads(false);
    auto v = values.unbind();
    ctx->mark_non_differentiable({v[1], v[2], logp});
    return {v[0], v[1], v[2], logp};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return variable_list(10);
    const auto held = ctx->saved_data.find("grad");
    TORCH_CHECK(held != ctx->saved_data.end(),
                "policy_loss_from_logits: its backward pass runs once (the gradient was handed "
                "over); use token_logprobs with policy_loss for several");
    Tensor grad = held->second.toTensor();
    ctx->saved_data.erase(held);
    return first_of(10, first_order("policy_loss_from_logits", [&] {
      scale_rows__op().call(grad, g[0], ctx->saved_data["scale"].toDouble());
      return grad;
    }));
  }
};

struct PreferenceLossFn : Function<PreferenceLossFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logp, const Tensor& offsets,
                               const optional<Tensor>& ref, const optional<Tensor>& mask,
                               double beta, double smoothing, int64_t kind, bool normalize) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [loss, rewards, slope] = preference_loss_op().call(logp, offsets, ref, mask, beta,
                                                            smoothing, kind, normalize);
    ctx->save_for_backward({slope, offsets, mask.has_value() ? *mask : Tensor()});
    ctx->saved_data["tokens"] = logp.numel();
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({rewards});
    return {loss, rewards};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return variable_list(8);
    const auto s = ctx->get_saved_variables();
    return first_of(8, first_order("preference_loss", [&] {
      return preference_grad_op().call(
          s[0], s[1], s[2].defined() ? optional<Tensor>(s[2]) : std::nullopt, g[0],
          ctx->saved_data["tokens"].toInt());
    }));
  }
};

bool records(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// A tangent would be lost where nothing is recorded: none of the functions has a
// forward-mode derivative, and says so.
void refuse_tangent(const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(/*level=*/0).defined(),
      name, ": forward-mode derivatives are not implemented");
}

// ---------------------------------------------------------------------------
// Checks
// ---------------------------------------------------------------------------
void check_device(const char* name, const Tensor& t, const Tensor& first) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, ": sinkslot_b200 runs on CUDA tensors only (got ",
                    t.device(), ")");
  TORCH_CHECK_VALUE(t.device() == first.device(), name, ": all tensors must be on one device");
}
void check_device(const char* name, const optional<Tensor>& t, const Tensor& first) {
  if (t.has_value()) check_device(name, *t, first);
}
void check_dtype(const char* name, const char* what, const Tensor& t) {
  const auto d = t.scalar_type();
  TORCH_CHECK_VALUE(d == at::kFloat || d == at::kHalf || d == at::kBFloat16, name, ": ", what,
                    " must be float32, float16 or bfloat16, got ", d);
}
void check_index(const char* name, const char* what, const Tensor& t) {
  const auto d = t.scalar_type();
  TORCH_CHECK_VALUE(d == at::kInt || d == at::kLong, name, ": ", what,
                    " must be int32 or int64, got ", d);
}
void check_constant(const char* name, const char* what, const Tensor& t) {
  refuse_tangent(name, t);
  TORCH_CHECK_VALUE(!records(t), name, ": no gradient is taken in ", what, "; detach it");
}
// One float32 value for each token, contiguous.
Tensor per_token(const char* name, const char* what, const Tensor& t, const Tensor& like) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, name, ": ", what, " must be float32, got ",
                    t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == like.sizes(), name, ": ", what, " must have the tokens' shape ",
                    like.sizes(), ", got ", t.sizes());
  return t.contiguous();
}
void check_packing(const char* name, const Tensor& like, optional<Tensor>& mask,
                   optional<Tensor>& offsets) {
  if (mask.has_value()) {
    TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool && mask->sizes() == like.sizes(), name,
                      ": mask must be bool of the tokens' shape ", like.sizes(), ", got ",
                      mask->scalar_type(), " ", mask->sizes());
    mask = mask->contiguous();
  }
  if (offsets.has_value()) {
    check_index(name, "offsets", *offsets);
    TORCH_CHECK_VALUE(offsets->dim() == 1 && offsets->numel() >= 2, name,
                      ": offsets must hold (sequences + 1) values, got ", offsets->sizes());
    offsets = offsets->contiguous();
  }
}
void check_logits(const char* name, const Tensor& logits, const Tensor& tokens,
                  double temperature) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, name,
                    ": logits need a vocabulary axis, got ", logits.sizes());
  TORCH_CHECK_VALUE(tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1), name,
                    ": tokens must have the shape ", logits.sizes().slice(0, logits.dim() - 1),
                    " of the logits' rows, got ", tokens.sizes());
  check_device(name, logits, logits);
  refuse_tangent(name, logits);
  check_device(name, tokens, logits);
  check_dtype(name, "logits", logits);
  check_index(name, "tokens", tokens);
  TORCH_CHECK_VALUE(temperature >= 1e-30 && temperature <= 1e30, name,
                    ": temperature must be in [1e-30, 1e30], got ", temperature);
  TORCH_CHECK_VALUE(tokens.numel() <= (int64_t(1) << 27), name,
                    ": more than 2^27 rows are not supported");
}
// Rows with contiguous elements.
Tensor unit_rows(const Tensor& t) {
  return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous();
}

struct PolicyInputs {
  Tensor old_logp, advantages;
  optional<Tensor> ref_logp, mask, offsets;
  PolicyArgs args;
};

PolicyInputs check_policy(const char* name, const Tensor& like, const Tensor& old_logp,
                          const Tensor& advantages, const optional<Tensor>& ref_logp,
                          const optional<Tensor>& mask, const optional<Tensor>& offsets,
                          double clip_low, double clip_high, double kl_coef, c10::string_view kl,
                          c10::string_view average) {
  check_device(name, like, like);
  refuse_tangent(name, like);  // (the log-probabilities, or whole-numbered tokens)
  check_device(name, old_logp, like);
  check_device(name, advantages, like);
  check_device(name, ref_logp, like);
  check_device(name, mask, like);
  check_device(name, offsets, like);
  check_constant(name, "old_logp", old_logp);
  check_constant(name, "advantages", advantages);
  if (ref_logp.has_value()) check_constant(name, "ref_logp", *ref_logp);
  PolicyInputs in{per_token(name, "old_logp", old_logp, like), advantages, ref_logp, mask,
                  offsets, {}};
  if (ref_logp.has_value()) in.ref_logp = per_token(name, "ref_logp", *ref_logp, like);
  check_packing(name, like, in.mask, in.offsets);
  const int64_t s = sequences(in.offsets);
  TORCH_CHECK_VALUE(advantages.scalar_type() == at::kFloat, name,
                    ": advantages must be float32, got ", advantages.scalar_type());
  const bool per = advantages.sizes() == like.sizes();
  TORCH_CHECK_VALUE(per || (advantages.dim() == 1 && advantages.numel() == s), name,
                    ": advantages must be one per token ", like.sizes(), " or per sequence [", s,
                    "], got ", advantages.sizes());
  in.advantages = advantages.contiguous();
  const int64_t k = kl == "k1" ? 1 : kl == "k2" ? 2 : kl == "k3" ? 3 : 0;
  TORCH_CHECK_VALUE(k, name, ": kl must be 'k1', 'k2' or 'k3', got '", kl, "'");
  TORCH_CHECK_VALUE(average == "token" || average == "sequence", name,
                    ": average must be 'token' or 'sequence', got '", average, "'");
  TORCH_CHECK_VALUE(clip_low >= 0.0 && clip_high >= 0.0, name,
                    ": clip_low and clip_high must be >= 0, got ", clip_low, ", ", clip_high);
  TORCH_CHECK_VALUE(std::isfinite(kl_coef), name, ": kl_coef must be finite, got ", kl_coef);
  TORCH_CHECK_VALUE(kl_coef == 0.0 || ref_logp.has_value(), name, ": kl_coef ", kl_coef,
                    " needs ref_logp");
  in.args = {per, clip_low, clip_high, kl_coef, k, average == "sequence"};
  return in;
}

// ---------------------------------------------------------------------------
// What users call (the Python functions of the same names)
// ---------------------------------------------------------------------------
Tensor embedding_lookup(const Tensor& table_, const Tensor& index, double scale,
                        optional<int64_t> padding_index) {
  const char* name = "embedding_lookup";
  TORCH_CHECK_VALUE(table_.dim() == 2 && table_.size(0) >= 1 && table_.size(1) >= 1, name,
                    ": table must be (rows, dim), got ", table_.sizes());
  check_device(name, table_, table_);
  refuse_tangent(name, table_);
  check_device(name, index, table_);
  check_dtype(name, "table", table_);
  check_index(name, "index", index);
  const int64_t rows = table_.size(0);
  TORCH_CHECK_VALUE(rows < (int64_t(1) << 31) && index.numel() < (int64_t(1) << 31), name,
                    ": 2^31 rows or tokens and more are not supported");
  int64_t padding = -1;
  if (padding_index.has_value()) {
    TORCH_CHECK_VALUE(*padding_index >= -rows && *padding_index < rows, name, ": padding_index ",
                      *padding_index, " is outside the table of ", rows, " rows");
    padding = *padding_index < 0 ? *padding_index + rows : *padding_index;
  }
  const Tensor table = unit_rows(table_);
  const Tensor flat = index.dim() == 1 && index.is_contiguous() ? index
                                                                : index.reshape({-1}).contiguous();
  Tensor out = records(table) ? LookupFn::apply(table, flat, scale, padding)
                              : lookup_op().call(table, flat, scale);
  if (index.dim() == 1) return out;
  auto shape = index.sizes().vec();
  shape.push_back(table.size(1));
  return out.view(shape);
}

std::tuple<Tensor, Tensor> logprobs(const Tensor& logits, const Tensor& tokens, double temperature,
                                    int64_t ignore_index, bool entropy) {
  const char* name = "token_logprobs";
  check_logits(name, logits, tokens, temperature);
  const Tensor z =
      unit_rows(logits.dim() == 2 ? logits : logits.reshape({-1, logits.size(-1)}));
  const Tensor flat = tokens.dim() == 1 && tokens.is_contiguous()
                          ? tokens
                          : tokens.reshape({-1}).contiguous();
  Tensor logp, ent;
  if (records(z)) {
    auto out = TokenLogprobsFn::apply(z, flat, temperature, ignore_index, entropy);
    logp = out[0];
    if (entropy) ent = out[1];
  } else {
    std::tie(logp, ent, std::ignore) =
        token_logprobs_op().call(z, flat, temperature, ignore_index, entropy);
  }
  if (tokens.dim() != 1) {
    logp = logp.view(tokens.sizes());
    if (entropy) ent = ent.view(tokens.sizes());
  }
  return {logp, entropy ? ent : logp};
}

std::tuple<Tensor, Tensor, Tensor> policy(const Tensor& logp, const Tensor& old_logp,
                                          const Tensor& advantages,
                                          const optional<Tensor>& ref_logp,
                                          const optional<Tensor>& mask,
                                          const optional<Tensor>& offsets, double clip_low,
                                          double clip_high, double kl_coef, c10::string_view kl,
                                          c10::string_view average) {
  const char* name = "policy_loss";
  TORCH_CHECK_VALUE(logp.dim() == 1, name, ": logp must be (tokens,), got ", logp.sizes());
  const PolicyInputs in = check_policy(name, logp, old_logp, advantages, ref_logp, mask, offsets,
                                       clip_low, clip_high, kl_coef, kl, average);
  const Tensor flat = per_token(name, "logp", logp, logp);
  if (records(flat)) {
    auto out = PolicyLossFn::apply(flat, in.old_logp, in.advantages, in.ref_logp, in.mask,
                                   in.offsets, in.args);
    return {out[0], out[1], out[2]};
  }
  const PolicyArgs& a = in.args;
  auto v = std::get<0>(policy_loss_op().call(flat, in.old_logp, in.advantages, in.ref_logp,
                                             in.mask, in.offsets, a.adv_per_token, a.clip_low,
                                             a.clip_high, a.kl_coef, a.kl, a.sequence_average,
                                             false))
               .unbind();
  return {v[0], v[1], v[2]};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> policy_from_logits(
    const Tensor& logits, const Tensor& tokens, const Tensor& old_logp, const Tensor& advantages,
    double temperature, const optional<Tensor>& ref_logp, const optional<Tensor>& mask,
    const optional<Tensor>& offsets, double clip_low, double clip_high, double kl_coef,
    c10::string_view kl, c10::string_view average, double grad_scale) {
  const char* name = "policy_loss_from_logits";
  TORCH_CHECK_VALUE(logits.dim() == 2, name, ": logits must be (tokens, vocab), got ",
                    logits.sizes());
  check_logits(name, logits, tokens, temperature);
  TORCH_CHECK_VALUE(std::isnormal((float)grad_scale), name,
                    ": grad_scale must be a normal float32, got ", grad_scale);
  const PolicyInputs in = check_policy(name, tokens, old_logp, advantages, ref_logp, mask, offsets,
                                       clip_low, clip_high, kl_coef, kl, average);
  const Tensor z = unit_rows(logits), flat = tokens.contiguous();
  const PolicyArgs& a = in.args;
  if (records(z)) {
    auto out = PolicyLossLogitsFn::apply(z, flat, in.old_logp, in.advantages, in.ref_logp, in.mask,
                                         in.offsets, temperature, a, grad_scale);
    return {out[0], out[1], out[2], out[3]};
  }
  auto [values, logp, none] = policy_loss_logits_op().call(
      z, flat, in.old_logp, in.advantages, in.ref_logp, in.mask, in.offsets, temperature,
      a.adv_per_token, a.clip_low, a.clip_high, a.kl_coef, a.kl, a.sequence_average, grad_scale,
      false);
  auto v = values.unbind();
  return {v[0], v[1], v[2], logp};
}

std::tuple<Tensor, Tensor> preference(const Tensor& logp, const Tensor& offsets_,
                                      const optional<Tensor>& ref_logp_,
                                      const optional<Tensor>& mask_, double beta, double smoothing,
                                      c10::string_view kind, bool normalize) {
  const char* name = "preference_loss";
  TORCH_CHECK_VALUE(logp.dim() == 1, name, ": logp must be (tokens,), got ", logp.sizes());
  check_device(name, logp, logp);
  refuse_tangent(name, logp);
  check_device(name, offsets_, logp);
  check_device(name, ref_logp_, logp);
  check_device(name, mask_, logp);
  if (ref_logp_.has_value()) check_constant(name, "ref_logp", *ref_logp_);
  const int64_t k = kind == "sigmoid" ? 0 : kind == "hinge" ? 1 : kind == "squared" ? 2 : -1;
  TORCH_CHECK_VALUE(k >= 0, name, ": kind must be 'sigmoid', 'hinge' or 'squared', got '", kind,
                    "'");
  TORCH_CHECK_VALUE(beta > 0.0 && std::isfinite(beta), name,
                    ": beta must be positive and finite, got ", beta);
  TORCH_CHECK_VALUE(smoothing >= 0.0 && smoothing < 1.0 && (smoothing == 0.0 || k == 0), name,
                    ": label_smoothing must be in [0, 1), and 0 unless kind is 'sigmoid'; got ",
                    smoothing);
  optional<Tensor> mask = mask_, offsets = offsets_, ref_logp = ref_logp_;
  check_packing(name, logp, mask, offsets);
  TORCH_CHECK_VALUE(offsets->numel() % 2 == 1, name, ": sequences come in pairs, got ",
                    offsets->numel() - 1);
  if (ref_logp.has_value()) ref_logp = per_token(name, "ref_logp", *ref_logp, logp);
  const Tensor flat = per_token(name, "logp", logp, logp);
  if (records(flat)) {
    auto out = PreferenceLossFn::apply(flat, *offsets, ref_logp, mask, beta, smoothing, k,
                                       normalize);
    return {out[0], out[1]};
  }
  auto [loss, rewards, slope] = preference_loss_op().call(flat, *offsets, ref_logp, mask, beta,
                                                          smoothing, k, normalize);
  return {loss, rewards};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sinkslot_b200, m) {
  m.def("lookup(Tensor table, Tensor index, float scale) -> Tensor");
  m.def("lookup_grad(Tensor grad_out, Tensor index, int rows, float scale, int padding) -> Tensor");
  m.def("token_logprobs(Tensor logits, Tensor tokens, float temperature, int ignore_index, "
        "bool entropy) -> (Tensor, Tensor, Tensor)");
  m.def("token_logprobs_grad(Tensor logits, Tensor tokens, Tensor stats, Tensor entropy, "
        "Tensor? g, Tensor? g_entropy, float temperature, int ignore_index) -> Tensor");
  m.def("policy_loss(Tensor logp, Tensor old_logp, Tensor advantages, Tensor? ref_logp, "
        "Tensor? mask, Tensor? offsets, bool adv_per_token, float clip_low, float clip_high, "
        "float kl_coef, int kl, bool sequence_average, bool want_grad) -> (Tensor, Tensor)");
  m.def("scale_tokens(Tensor coef, Tensor values, Tensor g) -> Tensor");
  m.def("policy_loss_logits(Tensor logits, Tensor tokens, Tensor old_logp, Tensor advantages, "
        "Tensor? ref_logp, Tensor? mask, Tensor? offsets, float temperature, bool adv_per_token, "
        "float clip_low, float clip_high, float kl_coef, int kl, bool sequence_average, "
        "float grad_scale, bool want_grad) -> (Tensor, Tensor, Tensor)");
  m.def("scale_rows_(Tensor(a!) grad, Tensor g, float grad_scale) -> ()");
  m.def("preference_loss(Tensor logp, Tensor offsets, Tensor? ref_logp, Tensor? mask, float beta, "
        "float smoothing, int kind, bool normalize) -> (Tensor, Tensor, Tensor)");
  m.def("preference_grad(Tensor slope, Tensor offsets, Tensor? mask, Tensor g, int tokens) "
        "-> Tensor");

  m.def("embedding_lookup(Tensor table, Tensor index, float scale=1.0, int? padding_index=None) "
        "-> Tensor", embedding_lookup);
  m.def("logprobs(Tensor logits, Tensor tokens, float temperature=1.0, int ignore_index=-100, "
        "bool entropy=False) -> (Tensor, Tensor)", logprobs);
  m.def("policy(Tensor logp, Tensor old_logp, Tensor advantages, Tensor? ref_logp, Tensor? mask, "
        "Tensor? offsets, float clip_low, float clip_high, float kl_coef, str kl, str average) "
        "-> (Tensor, Tensor, Tensor)", policy);
  m.def("policy_from_logits(Tensor logits, Tensor tokens, Tensor old_logp, Tensor advantages, "
        "float temperature, Tensor? ref_logp, Tensor? mask, Tensor? offsets, float clip_low, "
        "float clip_high, float kl_coef, str kl, str average, float grad_scale) "
        "-> (Tensor, Tensor, Tensor, Tensor)", policy_from_logits);
  m.def("preference(Tensor logp, Tensor offsets, Tensor? ref_logp, Tensor? mask, float beta, "
        "float label_smoothing, str kind, bool normalize) -> (Tensor, Tensor)", preference);
}

TORCH_LIBRARY_IMPL(sinkslot_b200, CUDA, m) {
  m.impl("lookup", lookup);
  m.impl("lookup_grad", lookup_grad);
  m.impl("token_logprobs", token_logprobs);
  m.impl("token_logprobs_grad", token_logprobs_grad);
  m.impl("policy_loss", policy_loss);
  m.impl("scale_tokens", scale_tokens);
  m.impl("policy_loss_logits", policy_loss_logits);
  m.impl("scale_rows_", scale_rows_);
  m.impl("preference_loss", preference_loss);
  m.impl("preference_grad", preference_grad);
}
