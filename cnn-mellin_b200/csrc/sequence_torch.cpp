// Torch binding of the sequence operators (gated recurrence, group norm with an activation, counter-based dropout):
// argument checks, allocation, the current stream and autograd around the C ABI in include/mellin_b200.h.  No kernels
// and no arithmetic here.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>
#include <torch/torch.h>

#include <string>
#include <tuple>
#include <vector>

#include "mellin_b200.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using OptTensor = c10::optional<Tensor>;

// the entry points of one storage type: P = what its pointers are declared as, S = what states and parameters are
#define SEQUENCE_API(NAME, SUFFIX, PT, ST)                                                     \
  struct NAME {                                                                                \
    using P = PT;                                                                              \
    using S = ST;                                                                              \
    static constexpr auto recurrence = mellin_gated_recurrence_##SUFFIX;                       \
    static constexpr auto recurrence_backward = mellin_gated_recurrence_backward_##SUFFIX;     \
    static constexpr auto norm = mellin_group_norm_act_##SUFFIX;                               \
    static constexpr auto norm_backward = mellin_group_norm_act_backward_##SUFFIX;             \
    static constexpr auto norm_workspace = mellin_group_norm_act_workspace_bytes_##SUFFIX;     \
    static constexpr auto dropout = mellin_philox_dropout_##SUFFIX;                            \
  };
SEQUENCE_API(ApiF32, f32, float, float)
SEQUENCE_API(ApiF64, f64, double, double)
SEQUENCE_API(ApiF16, f16, void, float)
SEQUENCE_API(ApiBF16, bf16, void, float)

template <typename F>
int by_type(at::ScalarType type, F &&f) {
  switch (type) {
    case at::kFloat: return f(ApiF32{});
    case at::kDouble: return f(ApiF64{});
    case at::kHalf: return f(ApiF16{});
    default: return f(ApiBF16{});
  }
}

template <typename P>
P *ptr(const Tensor &t) {
  return t.defined() && t.numel() > 0 ? static_cast<P *>(t.data_ptr()) : nullptr;
}

void check_status(int code, const char *op) {
  TORCH_CHECK(code == MELLIN_OK, "mellin_b200 error ", code, " in ", op, ": ", mellin_last_error());
}

void *current_stream(const Tensor &t) {
  return static_cast<void *>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

at::ScalarType state_type(const Tensor &t) { return t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }
// a state or parameter as the C ABI takes it
Tensor as_state(const Tensor &input, const OptTensor &p) {
  if (!p) return Tensor();
  return p->scalar_type() == state_type(input) && p->is_contiguous() ? *p : p->to(state_type(input)).contiguous();
}

// ---- checks ---------------------------------------------------------------------------------------------------------

void check_input(const char *c, const Tensor &t, const char *name) {
  TORCH_CHECK(t.is_cuda(), c, ": '", name, "' must be a CUDA tensor (this build has no CPU path)");
  TORCH_CHECK(t.layout() == at::kStrided, c, ": '", name, "' must be a dense tensor");
  const auto type = t.scalar_type();
  TORCH_CHECK(type == at::kFloat || type == at::kDouble || type == at::kHalf || type == at::kBFloat16, c, ": '", name,
              "' must be float16, bfloat16, float32 or float64, got ", type);
}

void check_like(const char *c, const Tensor &t, const char *name, const Tensor &input, at::IntArrayRef sizes) {
  check_input(c, t, name);
  TORCH_CHECK(t.device() == input.device(), c, ": '", name, "' must be on the same device as 'input'");
  TORCH_CHECK(t.sizes() == sizes, c, ": expected '", name, "' to have shape ", sizes, ", got ", t.sizes());
}

void check_same_type(const char *c, const Tensor &t, const char *name, const Tensor &input) {
  TORCH_CHECK(t.scalar_type() == input.scalar_type(), c, ": '", name, "' and 'input' must have the same dtype");
}

void check_lens(const char *c, const OptTensor &lens, const Tensor &input) {
  if (!lens) return;
  TORCH_CHECK(lens->is_cuda() && lens->scalar_type() == at::kInt && lens->dim() == 1 && lens->size(0) == input.size(0), c,
              ": 'lens' must be an int32 CUDA tensor with one length per utterance");
  TORCH_CHECK(lens->device() == input.device(), c, ": 'lens' must be on the same device as 'input'");
}

// ---- operands -------------------------------------------------------------------------------------------------------

// (batch, frames, channels) with adjacent channels; anything else is copied
Tensor frames_view(const Tensor &t) { return t.size(2) <= 1 || t.stride(2) == 1 ? t : t.contiguous(); }

// a new tensor whose frames lie as those of `like` do: utterance after utterance, or frame after frame (time-major)
Tensor empty_frames(const Tensor &like, int64_t channels) {
  const int64_t n = like.size(0), t = like.size(1);
  if (n > 1 && t > 1 && like.stride(0) < like.stride(1))
    return at::empty({t, n, channels}, like.options()).transpose(0, 1);
  return at::empty({n, t, channels}, like.options());
}

const int *lens_ptr(const OptTensor &lens) { return lens && lens->numel() > 0 ? lens->data_ptr<int>() : nullptr; }
OptTensor dense(const OptTensor &lens) { return lens && !lens->is_contiguous() ? OptTensor(lens->contiguous()) : lens; }

// gradients that a second differentiation would silently miss: refuse it when it comes to that
tensor_list once_differentiable(const char *what, tensor_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  std::vector<size_t> at;
  tensor_list defined;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) at.push_back(i), defined.push_back(grads[i].detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once only",
                                                               static_cast<int64_t>(defined.size()));
  auto marked = (*error)(std::move(defined));
  for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = marked[i];
  return grads;
}

// Whether a call is differentiated with regard to any of its operands.  Forward mode counts, which needs neither
// requires_grad nor grad mode: there is none here, and the autograd function says so, where its kernels alone would drop the
// tangents.
bool differentiated(const Tensor &t) {
  return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined();
}
bool differentiated(const OptTensor &t) { return t && differentiated(*t); }

// ---- gated recurrence -----------------------------------------------------------------------------------------------

// What the C ABI takes of a (batch, frames, channels) tensor, or of its channels from `first` on: no tensor is made for it
struct View {
  void *p = nullptr;
  int64_t sn = 0, st = 0;
  View() = default;
  explicit View(const Tensor &t, int64_t first = 0) {
    if (!t.defined() || t.numel() == 0) return;
    p = static_cast<char *>(t.data_ptr()) + first * t.element_size();
    sn = t.stride(0), st = t.stride(1);
  }
};

// (output, final state, states kept for backward)
std::tuple<Tensor, Tensor, Tensor> recurrence_forward(const Tensor &input, const OptTensor &gate, const OptTensor &initial,
                                                      const OptTensor &lens_in, bool reverse, bool keep_states) {
  const char *c = "gated_recurrence";
  check_input(c, input, "input");
  TORCH_CHECK(input.dim() == 3, c, ": expected 'input' to be (batch, frames, channels), got ", input.dim(), " dimensions");
  if (gate) {
    check_like(c, *gate, "gate", input, input.sizes());
    check_same_type(c, *gate, "gate", input);
  } else {
    TORCH_CHECK(input.size(2) % 2 == 0, c, ": without 'gate', 'input' holds values and gates: an even number of channels");
  }
  const int64_t n = input.size(0), t = input.size(1), channels = gate ? input.size(2) : input.size(2) / 2;
  if (initial) check_like(c, *initial, "initial", input, {n, channels});
  check_lens(c, lens_in, input);
  c10::cuda::CUDAGuard guard(input.device());
  const Tensor in = frames_view(input), gate_in = gate ? frames_view(*gate) : in;
  const View x(in), g(gate_in, gate ? 0 : channels);
  const OptTensor lens = dense(lens_in);
  const auto state_options = input.options().dtype(state_type(input));
  const Tensor h0 = as_state(input, initial);
  Tensor y = empty_frames(input, channels), final = at::empty({n, channels}, state_options), states;
  if (keep_states) states = at::empty({mellin_gated_recurrence_state_count(n, t, channels)}, state_options);
  check_status(by_type(input.scalar_type(), [&](auto api) {
    using A = decltype(api);
    using P = typename A::P;
    using S = typename A::S;
    return A::recurrence(static_cast<P *>(x.p), x.sn, x.st, static_cast<P *>(g.p), g.sn, g.st, ptr<S>(h0), lens_ptr(lens),
                         reverse ? 1 : 0, n, t, channels, ptr<P>(y), y.stride(0), y.stride(1), ptr<S>(final), ptr<S>(states), current_stream(input));
  }), c);
  return {y, final, states};
}

std::tuple<Tensor, Tensor> gated_recurrence_cuda(const Tensor &input, const OptTensor &gate, const OptTensor &initial,
                                                 const OptTensor &lens, bool reverse) {
  auto [y, final, states] = recurrence_forward(input, gate, initial, lens, reverse, false);
  return {y, final};
}

class GatedRecurrenceFunction : public torch::autograd::Function<GatedRecurrenceFunction> {
 public:
  static tensor_list forward(AutogradContext *ctx, const Tensor &input, const OptTensor &gate, const OptTensor &initial,
                             const OptTensor &lens, bool reverse) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, final, states] = recurrence_forward(input, gate, initial, lens, reverse, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({input, gate ? *gate : Tensor(), states, lens ? *lens : Tensor()});
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["initial"] = initial ? static_cast<int64_t>(initial->scalar_type()) : int64_t(-1);
    return {y, final};
  }
  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    const char *c = "gated_recurrence backward";
    auto saved = ctx->get_saved_variables();
    const Tensor &input = saved[0], &states = saved[2];
    const OptTensor gate = saved[1].defined() ? OptTensor(saved[1]) : OptTensor();
    const OptTensor lens = dense(saved[3].defined() ? OptTensor(saved[3]) : OptTensor());
    const int64_t initial_type = ctx->saved_data["initial"].toInt();
    Tensor gx, gg, gi;  // without a gate tensor, gx holds both gradients
    {
      at::AutoDispatchBelowADInplaceOrView below;
      c10::cuda::CUDAGuard guard(input.device());
      const Tensor in = frames_view(input), gate_in = gate ? frames_view(*gate) : in;
      const int64_t n = in.size(0), t = in.size(1), channels = gate ? in.size(2) : in.size(2) / 2;
      gx = empty_frames(input, in.size(2));
      if (gate) gg = empty_frames(*gate, channels);
      const View x(in), g(gate_in, gate ? 0 : channels), ox(gx), og(gate ? gg : gx, gate ? 0 : channels);
      const Tensor gy = grads[0].defined() ? frames_view(grads[0]) : Tensor();
      const Tensor gf = grads[1].defined() ? grads[1].contiguous() : Tensor();
      if (initial_type >= 0) gi = at::empty({n, channels}, input.options().dtype(state_type(input)));
      check_status(by_type(input.scalar_type(), [&](auto api) {
        using A = decltype(api);
        using P = typename A::P;
        using S = typename A::S;
        return A::recurrence_backward(
            static_cast<P *>(x.p), x.sn, x.st, static_cast<P *>(g.p), g.sn, g.st, ptr<S>(states), lens_ptr(lens),
            ctx->saved_data["reverse"].toBool() ? 1 : 0, n, t, channels, ptr<P>(gy), gy.defined() ? gy.stride(0) : 0,
            gy.defined() ? gy.stride(1) : 0, ptr<S>(gf), static_cast<P *>(ox.p), ox.sn, ox.st, static_cast<P *>(og.p), og.sn,
            og.st, ptr<S>(gi), current_stream(input));
      }), c);
      if (gi.defined() && static_cast<int64_t>(gi.scalar_type()) != initial_type)
        gi = gi.to(static_cast<at::ScalarType>(initial_type));
    }
    return once_differentiable("gated_recurrence", {gx, gg, gi, Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor> gated_recurrence_autograd(const Tensor &input, const OptTensor &gate, const OptTensor &initial,
                                                     const OptTensor &lens, bool reverse) {
  if (differentiated(input) || differentiated(gate) || differentiated(initial)) {
    auto out = GatedRecurrenceFunction::apply(input, gate, initial, lens, reverse);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return gated_recurrence_cuda(input, gate, initial, lens, reverse);
}

// ---- group norm with an activation ----------------------------------------------------------------------------------

// (output, statistics) of a (batch, frames, channels) tensor
std::tuple<Tensor, Tensor> norm_forward(const Tensor &input, int64_t groups, const OptTensor &weight, const OptTensor &bias,
                                        const OptTensor &lens_in, double eps, int64_t act, bool keep_stats) {
  const char *c = "group_norm_act";
  check_input(c, input, "input");
  TORCH_CHECK(input.dim() == 3, c, ": expected (batch, frames, channels)");
  const int64_t n = input.size(0), t = input.size(1), channels = input.size(2);
  TORCH_CHECK(groups > 0 && channels % groups == 0, c, ": ", channels, " channels do not divide into ", groups, " groups");
  TORCH_CHECK(eps >= 0, c, ": 'eps' must not be negative");
  TORCH_CHECK(act >= 0 && act <= 3, c, ": unknown activation ", act);
  if (weight) check_like(c, *weight, "weight", input, {channels});
  if (bias) check_like(c, *bias, "bias", input, {channels});
  check_lens(c, lens_in, input);
  c10::cuda::CUDAGuard guard(input.device());
  const Tensor x = frames_view(input), w = as_state(input, weight), b = as_state(input, bias);
  const OptTensor lens = dense(lens_in);
  Tensor y = empty_frames(input, channels), stats;
  if (keep_stats) stats = at::empty({n, groups, 2}, input.options().dtype(state_type(input)));
  check_status(by_type(input.scalar_type(), [&](auto api) {
    using A = decltype(api);
    using P = typename A::P;
    using S = typename A::S;
    const size_t bytes = A::norm_workspace(n, t, channels, groups, 0);
    const Tensor ws = bytes > 0 ? at::empty({static_cast<int64_t>(bytes)}, input.options().dtype(at::kByte)) : Tensor();
    return A::norm(ptr<P>(x), x.stride(0), x.stride(1), ptr<S>(w), ptr<S>(b), lens_ptr(lens), n, t, channels, groups, eps,
                   static_cast<int>(act), ptr<P>(y), y.stride(0), y.stride(1), ptr<S>(stats), ptr<void>(ws), bytes,
                   current_stream(input));
  }), c);
  return {y, stats};
}

class GroupNormActFunction : public torch::autograd::Function<GroupNormActFunction> {
 public:
  static Tensor forward(AutogradContext *ctx, const Tensor &input, int64_t groups, const OptTensor &weight,
                        const OptTensor &bias, const OptTensor &lens, double eps, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, stats] = norm_forward(input, groups, weight, bias, lens, eps, act, true);
    ctx->save_for_backward({input, weight ? *weight : Tensor(), bias ? *bias : Tensor(), lens ? *lens : Tensor(), stats});
    ctx->saved_data["groups"] = groups, ctx->saved_data["act"] = act;
    return y;
  }
  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    const char *c = "group_norm_act backward";
    auto saved = ctx->get_saved_variables();
    const Tensor &input = saved[0], &stats = saved[4];
    const OptTensor weight = saved[1].defined() ? OptTensor(saved[1]) : OptTensor();
    const OptTensor bias = saved[2].defined() ? OptTensor(saved[2]) : OptTensor();
    const OptTensor lens = dense(saved[3].defined() ? OptTensor(saved[3]) : OptTensor());
    Tensor gx, gw, gb;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      c10::cuda::CUDAGuard guard(input.device());
      const int64_t n = input.size(0), t = input.size(1), channels = input.size(2);
      const Tensor x = frames_view(input), gy = frames_view(grads[0]);
      const Tensor w = as_state(input, weight), b = as_state(input, bias);
      gx = empty_frames(input, channels);
      const auto options = input.options().dtype(state_type(input));
      if (weight) gw = at::empty({channels}, options);
      if (bias) gb = at::empty({channels}, options);
      check_status(by_type(input.scalar_type(), [&](auto api) {
        using A = decltype(api);
        using P = typename A::P;
        using S = typename A::S;
        const size_t bytes = A::norm_workspace(n, t, channels, ctx->saved_data["groups"].toInt(), 1);
        const Tensor ws = bytes > 0 ? at::empty({static_cast<int64_t>(bytes)}, input.options().dtype(at::kByte)) : Tensor();
        return A::norm_backward(ptr<P>(x), x.stride(0), x.stride(1), ptr<S>(w), ptr<S>(b), ptr<S>(stats), lens_ptr(lens), n,
                                t, channels, ctx->saved_data["groups"].toInt(),
                                static_cast<int>(ctx->saved_data["act"].toInt()), ptr<P>(gy), gy.stride(0), gy.stride(1),
                                ptr<P>(gx), gx.stride(0), gx.stride(1), ptr<S>(gw), ptr<S>(gb), ptr<void>(ws), bytes,
                                current_stream(input));
      }), c);
      if (weight && gw.scalar_type() != weight->scalar_type()) gw = gw.to(weight->scalar_type());
      if (bias && gb.scalar_type() != bias->scalar_type()) gb = gb.to(bias->scalar_type());
    }
    return once_differentiable("group_norm_act", {gx, Tensor(), gw, gb, Tensor(), Tensor(), Tensor()});
  }
};

// (batch, *, channels) as (batch, frames, channels)
Tensor as_frames(const char *c, const Tensor &input, const OptTensor &lens) {
  TORCH_CHECK(input.dim() >= 2, c, ": expected 'input' to be (batch, ..., channels), got ", input.dim(), " dimensions");
  TORCH_CHECK(!lens || input.dim() == 3, c, ": 'lens' goes with a (batch, frames, channels) input");
  if (input.dim() == 3) return input;
  int64_t frames = 1;
  for (int64_t i = 1; i + 1 < input.dim(); ++i) frames *= input.size(i);
  return input.reshape({input.size(0), frames, input.size(-1)});
}

Tensor group_norm_act_cuda(const Tensor &input, int64_t groups, const OptTensor &weight, const OptTensor &bias,
                           const OptTensor &lens, double eps, int64_t act) {
  auto [y, stats] = norm_forward(as_frames("group_norm_act", input, lens), groups, weight, bias, lens, eps, act, false);
  return input.dim() == 3 ? y : y.reshape(input.sizes());
}

Tensor group_norm_act_autograd(const Tensor &input, int64_t groups, const OptTensor &weight, const OptTensor &bias,
                               const OptTensor &lens, double eps, int64_t act) {
  if (differentiated(input) || differentiated(weight) || differentiated(bias)) {
    const Tensor y = GroupNormActFunction::apply(as_frames("group_norm_act", input, lens), groups, weight, bias, lens, eps, act);
    return input.dim() == 3 ? y : y.reshape(input.sizes());
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return group_norm_act_cuda(input, groups, weight, bias, lens, eps, act);
}

// ---- counter-based dropout ------------------------------------------------------------------------------------------

// a tensor as rows of adjacent elements with one stride between them, in row-major order
struct Rows {
  Tensor t;
  int64_t rows = 1, cols = 0, stride = 0;
};
Rows as_rows(const Tensor &in) {
  if (in.is_contiguous() || in.dim() == 0 || in.numel() == 0) return {in, 1, in.numel(), in.numel()};
  bool regular = in.stride(-1) == 1;
  int64_t stride = in.dim() >= 2 ? in.stride(-2) : 0;
  for (int64_t i = in.dim() - 2; i > 0 && regular; --i) regular = in.stride(i - 1) == in.stride(i) * in.size(i);
  if (in.dim() < 2 || !regular) return {in.contiguous(), 1, in.numel(), in.numel()};
  return {in, in.numel() / in.size(-1), in.size(-1), stride};
}

Tensor dropout_pass(const char *c, const Tensor &input, double p, int64_t seed, const OptTensor &seed_tensor,
                    const OptTensor &residual) {
  c10::cuda::CUDAGuard guard(input.device());
  Tensor y = at::empty(input.sizes(), input.options());
  Rows x = as_rows(input), r;
  if (residual) r = as_rows(*residual);
  // rows of both the same length: a dense operand can be cut into the other's rows
  const int64_t cols = residual ? std::min(x.cols, r.cols) : x.cols;
  auto stride_of = [&](const Rows &v) { return v.cols == cols ? v.stride : cols; };
  const int64_t rows = cols > 0 ? input.numel() / cols : 0;
  check_status(by_type(input.scalar_type(), [&](auto api) {
    using A = decltype(api);
    using P = typename A::P;
    return A::dropout(ptr<P>(x.t), stride_of(x), residual ? ptr<P>(r.t) : nullptr, residual ? stride_of(r) : 0, rows, cols,
                      p, static_cast<uint64_t>(seed), seed_tensor ? seed_tensor->data_ptr<int64_t>() : nullptr, ptr<P>(y),
                      current_stream(input));
  }), c);
  return y;
}

void check_dropout(const Tensor &input, double p, const OptTensor &seed_tensor, const OptTensor &residual) {
  const char *c = "philox_dropout";
  check_input(c, input, "input");
  TORCH_CHECK(p >= 0.0 && p <= 1.0, c, ": 'p' must be in [0, 1], got ", p);
  if (seed_tensor)
    TORCH_CHECK(seed_tensor->is_cuda() && seed_tensor->scalar_type() == at::kLong && seed_tensor->numel() == 1 &&
                    seed_tensor->device() == input.device(),
                c, ": a seed tensor must be one int64 value on the device of 'input'");
  if (residual) {
    check_like(c, *residual, "residual", input, input.sizes());
    check_same_type(c, *residual, "residual", input);
  }
}

Tensor philox_dropout_cuda(const Tensor &input, double p, int64_t seed, const OptTensor &seed_tensor,
                           const OptTensor &residual) {
  check_dropout(input, p, seed_tensor, residual);
  return dropout_pass("philox_dropout", input, p, seed, seed_tensor, residual);
}

class PhiloxDropoutFunction : public torch::autograd::Function<PhiloxDropoutFunction> {
 public:
  static Tensor forward(AutogradContext *ctx, const Tensor &input, double p, int64_t seed, const OptTensor &seed_tensor,
                        const OptTensor &residual) {
    at::AutoDispatchBelowADInplaceOrView guard;
    // a seed tensor that is overwritten before backward would change the mask: autograd's version check refuses it
    ctx->save_for_backward({seed_tensor ? *seed_tensor : Tensor()});
    ctx->saved_data["p"] = p, ctx->saved_data["seed"] = seed, ctx->saved_data["residual"] = residual.has_value();
    return philox_dropout_cuda(input, p, seed, seed_tensor, residual);
  }
  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    auto saved = ctx->get_saved_variables();
    const OptTensor seed_tensor = saved[0].defined() ? OptTensor(saved[0]) : OptTensor();
    Tensor gx;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      gx = dropout_pass("philox_dropout backward", grads[0], ctx->saved_data["p"].toDouble(),
                        ctx->saved_data["seed"].toInt(), seed_tensor, OptTensor());
    }
    gx = once_differentiable("philox_dropout", {gx})[0];
    return {gx, Tensor(), Tensor(), Tensor(), ctx->saved_data["residual"].toBool() ? grads[0] : Tensor()};
  }
};

Tensor philox_dropout_autograd(const Tensor &input, double p, int64_t seed, const OptTensor &seed_tensor,
                               const OptTensor &residual) {
  if (differentiated(input) || differentiated(residual))
    return PhiloxDropoutFunction::apply(input, p, seed, seed_tensor, residual);
  at::AutoDispatchBelowADInplaceOrView guard;
  return philox_dropout_cuda(input, p, seed, seed_tensor, residual);
}

// ---- autocast: operands that autocast left in different types meet in the wider one -------------------------------

std::tuple<Tensor, OptTensor> widest(const Tensor &a, const OptTensor &b) {
  if (!b || a.scalar_type() == b->scalar_type() || !a.is_floating_point() || !b->is_floating_point()) return {a, b};
  const auto type = at::promote_types(a.scalar_type(), b->scalar_type());
  return {a.to(type), OptTensor(b->to(type))};
}

std::tuple<Tensor, Tensor> gated_recurrence_autocast(const Tensor &input, const OptTensor &gate, const OptTensor &initial,
                                                     const OptTensor &lens, bool reverse) {
  c10::impl::ExcludeDispatchKeyGuard below(c10::DispatchKey::Autocast);
  auto [x, g] = widest(input, gate);
  return c10::Dispatcher::singleton()
      .findSchemaOrThrow("mellin::gated_recurrence", "")
      .typed<std::tuple<Tensor, Tensor>(const Tensor &, const OptTensor &, const OptTensor &, const OptTensor &, bool)>()
      .call(x, g, initial, lens, reverse);
}

Tensor philox_dropout_autocast(const Tensor &input, double p, int64_t seed, const OptTensor &seed_tensor,
                               const OptTensor &residual) {
  c10::impl::ExcludeDispatchKeyGuard below(c10::DispatchKey::Autocast);
  auto [x, r] = widest(input, residual);
  return c10::Dispatcher::singleton()
      .findSchemaOrThrow("mellin::philox_dropout", "")
      .typed<Tensor(const Tensor &, double, int64_t, const OptTensor &, const OptTensor &)>()
      .call(x, p, seed, seed_tensor, r);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mellin, m) {
  m.def("gated_recurrence(Tensor input, Tensor? gate=None, Tensor? initial=None, Tensor? lens=None, bool reverse=False) -> (Tensor, Tensor)");
  m.def("group_norm_act(Tensor input, int groups, Tensor? weight=None, Tensor? bias=None, Tensor? lens=None, float eps=1e-05, int act=0) -> Tensor");
  m.def("philox_dropout(Tensor input, float p, int seed, Tensor? seed_tensor=None, Tensor? residual=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(mellin, CUDA, m) {
  m.impl("gated_recurrence", gated_recurrence_cuda);
  m.impl("group_norm_act", group_norm_act_cuda);
  m.impl("philox_dropout", philox_dropout_cuda);
}

TORCH_LIBRARY_IMPL(mellin, Autocast, m) {
  m.impl("gated_recurrence", gated_recurrence_autocast);
  m.impl("philox_dropout", philox_dropout_autocast);
}

TORCH_LIBRARY_IMPL(mellin, Autograd, m) {
  m.impl("gated_recurrence", gated_recurrence_autograd);
  m.impl("group_norm_act", group_norm_act_autograd);
  m.impl("philox_dropout", philox_dropout_autograd);
}
