// The losses over the vocabulary as functions of torch's autograd: allocation, the library's calls (e4b_amd.h) on the
// current stream of the logits' device, and the graph between them.
//
// A backward pass runs on autograd's own thread of the device. With the functions here it needs no interpreter lock there:
// in Python the two threads hand the lock and its objects' cache lines back and forth, and a small call's forward and
// backward took 105 us of host time, of which torch's own engine is about 45.
#include <ATen/functorch/BatchedTensorImpl.h>
// behind the one above, whose own calls it would make ambiguous
#include <ATen/LegacyBatchedTensorImpl.h>
#include <c10/core/InferenceMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "e4b_amd.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

void check(const char* fn, int status) {
  if (status != E4B_OK)
    throw std::runtime_error(std::string(fn) + " failed with status " + std::to_string(status) + ": " + e4b_last_error());
}

int32_t dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kBFloat16: return E4B_BF16;
    case torch::kHalf: return E4B_FP16;
    case torch::kFloat: return E4B_FP32;
    default: throw std::invalid_argument("unsupported dtype");
  }
}

template <class T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

void on_device(std::initializer_list<Tensor> all, const Tensor& z) {
  for (const Tensor& t : all)
    if (t.defined() && t.device() != z.device()) throw std::invalid_argument("the losses' tensors are on different devices");
  if (!z.is_cuda()) throw std::invalid_argument("the MI355X kernels need tensors on the HIP device");
}

// Logits [seqs, tokens, vocab] with a contiguous last axis; labels int64 [seqs, tokens], mask bool [tokens] or [seqs, tokens],
// both contiguous or undefined.
e4b_logits describe(const Tensor& z, const Tensor& labels, const Tensor& mask, double temperature) {
  e4b_logits d{};
  d.logits = z.data_ptr();
  d.dtype = dtype_code(z);
  d.temperature = static_cast<float>(temperature);
  d.seqs = z.size(0);
  d.tokens = z.size(1);
  d.vocab = z.size(2);
  d.seq_stride = z.stride(0);
  d.row_stride = z.stride(1);
  d.labels = ptr<const int64_t>(labels);
  d.mask = ptr<const uint8_t>(mask);
  d.mask_stride = mask.defined() && mask.dim() == 2 ? d.tokens : 0;
  return d;
}

// A forward's workspace, where it needs one.
Tensor workspace_of(e4b_logits& d, const Tensor& z) {
  d.workspace_bytes = e4b_loss_workspace_bytes(&d);
  if (!d.workspace_bytes) return Tensor();
  Tensor ws = at::empty({static_cast<int64_t>(d.workspace_bytes)}, z.options().dtype(torch::kByte));
  d.workspace = ws.data_ptr();
  return ws;
}

hipStream_t stream_of(const Tensor& z) { return c10::hip::getCurrentHIPStream(z.device().index()).stream(); }

Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(torch::kFloat)); }

Tensor or_undefined(const Maybe& t) { return t ? *t : Tensor(); }

// What a graph may save of a tensor made in inference mode (sampled tokens, a teacher's entries): a copy.
Tensor keepable(const Tensor& t) {
  return t.defined() && t.is_inference() && !c10::InferenceMode::is_enabled() ? t.clone() : t;
}

// What a backward needs beside the tensors it saves: (logits, labels, mask, index, share, saved).
struct Kept {
  double temperature = 1.0;
  int64_t reduction = E4B_REDUCE_NONE;
  int64_t coef = 0;  // floats of coef behind the statistics: 0, one per sequence (1) or per token (2)
};

void keep(AutogradContext* ctx, const Kept& k) {
  ctx->saved_data["k"] = c10::IValue(std::make_tuple(k.temperature, k.reduction, k.coef));
}

// Whether torch's operators are recorded or stood in for (make_fx): what a kernel writes is not among them.
bool recorded() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  if (!Modes::any_modes_set()) return false;
  return Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL);
}

template <class F>
Tensor of_each(const Tensor& grad, const F& f);

// f of each slice all[i]
template <class F>
Tensor stack_of(const Tensor& all, const F& f) {
  std::vector<Tensor> out;
  for (int64_t i = 0; i < all.size(0); ++i) out.push_back(of_each(all.select(0, i), f));
  return at::stack(out);
}

// f(grad); where torch hands over several gradients as one, f of each: the kernels read memory. A vectorised Jacobian
// (is_grads_batched) and torch.func.vmap wrap them in two different ways.
template <class F>
Tensor of_each(const Tensor& grad, const F& f) {
  if (const auto* batch = at::functorch::maybeGetBatchedImpl(grad))
    return at::functorch::makeBatched(stack_of(batch->value().movedim(batch->bdim(), 0), f), 0, batch->level());
  if (const auto* batch = at::maybeGetBatchedImpl(grad)) {
    std::vector<int64_t> from, to, sizes;
    at::BatchDims dims;
    for (const at::BatchDim& b : batch->bdims()) {
      from.push_back(b.dim());
      sizes.push_back(batch->value().size(b.dim()));
      to.push_back(static_cast<int64_t>(to.size()));
      dims.emplace_back(b.level(), to.back());
    }
    const Tensor out = stack_of(batch->value().movedim(from, to).flatten(0, to.back()), f);
    return at::makeBatched(out.unflatten(0, sizes), dims);
  }
  // followed by forward-mode differentiation: f is linear
  if (const Tensor tangent = grad._fw_grad(0); tangent.defined())
    return at::_make_dual(f(grad._fw_primal(0)), f(tangent), 0);
  return f(grad);
}

Tensor backward_of(AutogradContext* ctx, const Tensor& upstream) {
  if (!upstream.defined()) return Tensor();
  if (at::GradMode::is_enabled())
    throw std::runtime_error("the losses over logits are differentiable once: no create_graph=True on the device");
  if (recorded())
    throw std::runtime_error("the losses' backward on the device cannot be recorded by itself: record the forward with it");
  const auto t = ctx->get_saved_variables();
  const Tensor &z = t[0], &labels = t[1], &mask = t[2], &index = t[3], &share = t[4], &saved = t[5];
  const auto k = ctx->saved_data["k"].toTuple();
  const double temperature = k->elements()[0].toDouble();
  const int64_t reduction = k->elements()[1].toInt(), coef = k->elements()[2].toInt();
  on_device({labels, mask, index, share, saved, upstream}, z);
  const c10::OptionalDeviceGuard guard(z.device());
  const e4b_logits d = describe(z, labels, mask, temperature);
  const int64_t rows = d.seqs * d.tokens;
  float* at = ptr<float>(saved);
  float* behind = at + 4 * rows;
  const int64_t coef_strides[2] = {coef == 2 ? d.tokens : 1, coef == 2 ? 1 : 0};
  const float* coef_at = coef ? behind : nullptr;
  if (coef == 2) behind += rows;
  // the means' factors, where the loss is one of means over tokens
  const bool means = reduction != E4B_REDUCE_NONE && coef != 1;
  return of_each(upstream, [&](const Tensor& one) {
    // complex products' backwards pass tensors whose memory holds their negative; zeros may come without memory
    const Tensor grad = one._is_zerotensor() ? at::zeros(one.sizes(), one.options()) : one.resolve_neg();
    const Tensor out = at::empty(z.sizes(), z.options().memory_format(c10::MemoryFormat::Contiguous));
    const int64_t grad_strides[2] = {grad.dim() > 0 ? grad.stride(0) : 0, grad.dim() > 1 ? grad.stride(1) : 0};
    check("e4b_loss_backward",
          e4b_loss_backward(&d, at, ptr<const float>(grad), grad.dim() > 0 ? grad.size(0) : 1, grad_strides, coef_at,
                            coef_strides, means ? behind : nullptr, reduction == E4B_REDUCE_SEQUENCE, ptr<const int64_t>(index),
                            ptr<const float>(share), index.defined() ? static_cast<int32_t>(index.size(2)) : 0, out.data_ptr(),
                            stream_of(z)));
    return out;
  });
}

// An empty loss of the reduction's shape, and the number of its means.
std::pair<Tensor, int64_t> reduced(const Tensor& z, int64_t reduction) {
  if (reduction == E4B_REDUCE_NONE) return {floats({z.size(0), z.size(1)}, z), 0};
  if (reduction == E4B_REDUCE_SEQUENCE) return {floats({z.size(0)}, z), z.size(0)};
  return {floats({}, z), 1};
}

struct Logprobs : Function<Logprobs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& labels, const Maybe& mask_, double temperature,
                        bool graph) {
    const Tensor mask = or_undefined(mask_);
    on_device({labels, mask}, z);
    const c10::OptionalDeviceGuard guard(z.device());
    e4b_logits d = describe(z, labels, mask, temperature);
    const Tensor workspace = workspace_of(d, z);
    const Tensor logps = floats({d.seqs, d.tokens}, z);
    Tensor saved;
    if (graph) saved = floats({4 * d.seqs * d.tokens}, z);
    check("e4b_token_logprobs", e4b_token_logprobs(&d, ptr<float>(logps), ptr<float>(saved), stream_of(z)));
    if (graph) {
      ctx->save_for_backward({z, keepable(labels), keepable(mask), Tensor(), Tensor(), saved});
      keep(ctx, {temperature, E4B_REDUCE_NONE, 0});
      ctx->set_materialize_grads(false);
    }
    return logps;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return {backward_of(ctx, g[0]), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

int32_t reference_kind(const Tensor& ref) {
  if (!ref.defined()) return E4B_REF_SEQUENCE;
  const bool wide = ref.scalar_type() == torch::kDouble;
  if (ref.dim() == 2) return wide ? E4B_REF_TOKEN_FP64 : E4B_REF_TOKEN;
  return wide ? E4B_REF_SEQUENCE_FP64 : E4B_REF_SEQUENCE;
}

struct Preference : Function<Preference> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& labels, const Maybe& mask_,
                               const Maybe& ref_, int64_t kind, double beta, double smoothing, bool average) {
    const Tensor mask = or_undefined(mask_), ref = or_undefined(ref_);
    on_device({labels, mask, ref}, z);
    const c10::OptionalDeviceGuard guard(z.device());
    e4b_logits d = describe(z, labels, mask, 1.0);
    const Tensor workspace = workspace_of(d, z);
    const int64_t rows = d.seqs * d.tokens;
    const Tensor loss = floats({d.seqs / 2}, z), rewards = floats({d.seqs}, z), saved = floats({4 * rows + d.seqs}, z);
    float* at = ptr<float>(saved);
    check("e4b_preference_loss",
          e4b_preference_loss(&d, ptr<const void>(ref), reference_kind(ref), static_cast<int32_t>(kind),
                              static_cast<float>(beta), static_cast<float>(smoothing), average, ptr<float>(loss),
                              ptr<float>(rewards), at, at + 4 * rows, stream_of(z)));
    ctx->save_for_backward({z, keepable(labels), keepable(mask), Tensor(), Tensor(), saved});
    keep(ctx, {1.0, E4B_REDUCE_SEQUENCE, 1});
    ctx->mark_non_differentiable({rewards});
    ctx->set_materialize_grads(false);
    return {loss, rewards};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(8);
    out[0] = backward_of(ctx, g[0]);
    return out;
  }
};

struct Policy : Function<Policy> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& labels, const Maybe& mask_,
                               const Tensor& old, const Tensor& advantages, const Maybe& ref_, double clip_lo, double clip_hi,
                               double kl_coef, double temperature, int64_t reduction) {
    const Tensor mask = or_undefined(mask_), ref = or_undefined(ref_);
    on_device({labels, mask, old, advantages, ref}, z);
    const c10::OptionalDeviceGuard guard(z.device());
    e4b_logits d = describe(z, labels, mask, temperature);
    const Tensor workspace = workspace_of(d, z);
    const int64_t rows = d.seqs * d.tokens;
    const auto [loss, means] = reduced(z, reduction);
    const Tensor logps = floats({d.seqs, d.tokens}, z), saved = floats({5 * rows + means + (means ? rows : 0)}, z);
    float *at = ptr<float>(saved), *coef = at + 4 * rows, *inv = coef + rows;
    check("e4b_policy_loss",
          e4b_policy_loss(&d, ptr<const float>(old), ptr<const float>(advantages), advantages.dim() == 2, ptr<const float>(ref),
                          static_cast<float>(clip_lo), static_cast<float>(clip_hi), static_cast<float>(kl_coef),
                          static_cast<int32_t>(reduction), ptr<float>(logps), means ? inv + means : ptr<float>(loss), at, coef,
                          ptr<float>(loss), inv, stream_of(z)));
    ctx->save_for_backward({z, keepable(labels), keepable(mask), Tensor(), Tensor(), saved});
    keep(ctx, {temperature, reduction, 2});
    ctx->mark_non_differentiable({logps});
    ctx->set_materialize_grads(false);
    return {loss, logps};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(11);
    out[0] = backward_of(ctx, g[0]);
    return out;
  }
};

struct Distill : Function<Distill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Maybe& mask_, const Tensor& teacher, const Tensor& index,
                        double temperature, int64_t reduction) {
    const Tensor mask = or_undefined(mask_);
    on_device({mask, teacher, index}, z);
    const c10::OptionalDeviceGuard guard(z.device());
    e4b_logits d = describe(z, Tensor(), mask, temperature);
    const Tensor workspace = workspace_of(d, z);
    const int64_t rows = d.seqs * d.tokens;
    const auto [loss, means] = reduced(z, reduction);
    const Tensor share = floats(index.sizes(), z), saved = floats({4 * rows + means + (means ? rows : 0)}, z);
    float *at = ptr<float>(saved), *inv = at + 4 * rows;
    check("e4b_distill_loss",
          e4b_distill_loss(&d, teacher.data_ptr(), dtype_code(teacher), ptr<const int64_t>(index),
                           static_cast<int32_t>(index.size(2)), static_cast<int32_t>(reduction), ptr<float>(share),
                           means ? inv + means : ptr<float>(loss), at, ptr<float>(loss), inv, stream_of(z)));
    ctx->save_for_backward({z, Tensor(), keepable(mask), keepable(index), share, saved});
    keep(ctx, {temperature, reduction, 0});
    ctx->set_materialize_grads(false);
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(6);
    out[0] = backward_of(ctx, g[0]);
    return out;
  }
};

Tensor token_logprobs(const Tensor& z, const Tensor& labels, const Maybe& mask, double temperature) {
  return Logprobs::apply(z, labels, mask, temperature, z.requires_grad() && at::GradMode::is_enabled());
}

std::tuple<Tensor, Tensor> preference_loss(const Tensor& z, const Tensor& labels, const Maybe& mask, const Maybe& ref,
                                           int64_t kind, double beta, double smoothing, bool average) {
  const auto o = Preference::apply(z, labels, mask, ref, kind, beta, smoothing, average);
  return {o[0], o[1]};
}

std::tuple<Tensor, Tensor> policy_loss(const Tensor& z, const Tensor& labels, const Maybe& mask, const Tensor& old,
                                       const Tensor& advantages, const Maybe& ref, double clip_lo, double clip_hi,
                                       double kl_coef, double temperature, int64_t reduction) {
  const auto o = Policy::apply(z, labels, mask, old, advantages, ref, clip_lo, clip_hi, kl_coef, temperature, reduction);
  return {o[0], o[1]};
}

Tensor distill_loss(const Tensor& z, const Maybe& mask, const Tensor& teacher, const Tensor& index, double temperature,
                    int64_t reduction) {
  return Distill::apply(z, mask, teacher, index, temperature, reduction);
}

}  // namespace

PYBIND11_MODULE(libe4b_torch, m) {
  m.def("token_logprobs", &token_logprobs);
  m.def("preference_loss", &preference_loss);
  m.def("policy_loss", &policy_loss);
  m.def("distill_loss", &distill_loss);
}
