// The transformer operators as differentiable calls on GPU tensors.  Checked and
// recorded here and not in Python: a pass over a few MB takes the GPU some 15 us, one
// over a token 3, and a Python function forward and backward takes 40 and more.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/hip/HIPGraphsC10Utils.h>

#include <initializer_list>
#include <vector>

std::vector<torch::Tensor> rms_norm_fwd(torch::Tensor x, torch::Tensor weight, c10::optional<torch::Tensor> residual,
                                        double eps, int64_t group, at::IntArrayRef shape);
std::vector<torch::Tensor> rms_norm_bwd(torch::Tensor dy, c10::optional<torch::Tensor> dsum, torch::Tensor s,
                                        torch::Tensor weight, torch::Tensor inv);
std::vector<torch::Tensor> rotary_turn(torch::Tensor q, c10::optional<torch::Tensor> k, torch::Tensor positions,
                                       torch::Tensor frequencies, bool interleaved, double amplitude, bool backward);
std::vector<torch::Tensor> attention_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, double scale, double softcap,
                                         c10::optional<torch::Tensor> slopes, bool causal,
                                         c10::optional<torch::Tensor> prefix, c10::optional<torch::Tensor> q_doc,
                                         c10::optional<torch::Tensor> k_doc, bool keep_rest);
std::vector<torch::Tensor> attention_bwd(torch::Tensor dout, torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                         torch::Tensor o, torch::Tensor lse, torch::Tensor rest, double scale, double softcap,
                                         c10::optional<torch::Tensor> slopes, bool causal,
                                         c10::optional<torch::Tensor> prefix, c10::optional<torch::Tensor> q_doc,
                                         c10::optional<torch::Tensor> k_doc);

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

OptTensor opt(const Tensor& x) { return x.defined() ? OptTensor(x) : c10::nullopt; }

void once(const char* name) {  // under create_graph=True the engine records what a backward does
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " is differentiable once: its gradient has no gradient");
}

// A leaf whose gradient is still to be added to by a living eager graph has that graph's
// stream; a captured backward pass would wait across to it, and instantiating such a graph
// ends the process.
void capturable(std::initializer_list<OptTensor> leaves, const char* name) {
  if (!at::GradMode::is_enabled() || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const auto& x : leaves) {
    if (!x.has_value() || !x->requires_grad() || !x->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*x);
    const auto stream = node ? node->stream() : c10::nullopt;
    TORCH_CHECK(!stream.has_value() || stream->id() == at::hip::getCurrentHIPStream(x->device().index()).id(), name,
                ": captured while an eager graph of the same leaf lives on another stream: drop its outputs first");
  }
}

Tensor rows(const Tensor& x) {
  if (x.dim() == 2 && x.is_contiguous()) return x;
  return x.reshape({x.size(-1) > 0 ? x.numel() / x.size(-1) : 0, x.size(-1)}).contiguous();
}

Tensor shaped(const Tensor& x, at::IntArrayRef sizes) { return x.sizes() == sizes ? x : x.view(sizes); }

bool floating(const Tensor& x) {
  return x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf;
}

void check_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384, "rms_norm: 1 to 16384 columns expected, got shape ", x.sizes());
  TORCH_CHECK_TYPE(floating(x), "rms_norm: fp32, bf16 or fp16 expected, got ", x.scalar_type());
  TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1), "rms_norm: weight ", weight.sizes(), " does not fit rows of ", x.size(-1));
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, "rms_norm: weight is ",
                   weight.scalar_type(), ", x is ", x.scalar_type());
  TORCH_CHECK_VALUE(weight.device() == x.device(), "rms_norm: tensors on ", x.device(), " and ", weight.device());
  if (residual.has_value()) {
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), "rms_norm: residual ", residual->sizes(),
                      " ", residual->scalar_type(), " does not match x ", x.sizes(), " ", x.scalar_type());
    TORCH_CHECK_VALUE(residual->device() == x.device(), "rms_norm: tensors on ", x.device(), " and ", residual->device());
  }
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
    const Tensor w = weight.contiguous();
    // made in their shape: a view from within a function may not be changed in place
    auto got = rms_norm_fwd(rows(x), w, residual.has_value() ? OptTensor(rows(*residual)) : c10::nullopt, eps, -1, x.sizes());
    variable_list out{got[0]};
    if (residual.has_value()) out.push_back(got[2]);
    ctx->save_for_backward({residual.has_value() ? out[1] : x, w, got[1]});
    ctx->saved_data["residual"] = residual.has_value();
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("rms_norm");
    const auto saved = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    const Tensor dsum = residual ? grads[1] : Tensor();
    if (!grads[0].defined()) return {dsum, Tensor(), dsum, Tensor()};  // only the sum was used
    auto got = rms_norm_bwd(rows(grads[0]), dsum.defined() ? OptTensor(rows(dsum)) : c10::nullopt, rows(saved[0]), saved[1], saved[2]);
    const Tensor dx = shaped(got[0], saved[0].sizes());
    return {dx, got[1], residual ? dx : Tensor(), Tensor()};
  }
};

Tensor last_stride_one(const Tensor& x) { return x.stride(-1) == 1 ? x : x.contiguous(); }

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& positions,
                               const Tensor& frequencies, bool interleaved, double amplitude) {
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["amplitude"] = amplitude;
    ctx->set_materialize_grads(false);
    return rotary_turn(last_stride_one(q), k.has_value() ? OptTensor(last_stride_one(*k)) : c10::nullopt, positions, frequencies,
                       interleaved, amplitude, false);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("rotary");
    const auto saved = ctx->get_saved_variables();
    variable_list out(6);
    std::vector<size_t> which;
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined()) which.push_back(i);
    if (which.empty()) return out;
    auto got = rotary_turn(last_stride_one(grads[which[0]]), which.size() > 1 ? OptTensor(last_stride_one(grads[which[1]])) : c10::nullopt,
                           saved[0], saved[1], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["amplitude"].toDouble(), true);
    for (size_t i = 0; i < which.size(); ++i) out[which[i]] = got[i];
    return out;
  }
};

// Rows as the attention kernels read them: `width` wide (zeros behind), 16-byte
// borders, under 16 MB apart (offsets within a tile are 32 bits).
Tensor ready(const Tensor& x, int64_t width) {
  if (x.size(3) != width) {  // not torch's padding, which keeps an order of dimensions where it knows one
    Tensor out = at::zeros({x.size(0), x.size(1), x.size(2), width}, x.options());
    out.narrow(3, 0, x.size(3)).copy_(x);
    return out;
  }
  const int64_t size = x.element_size(), per16 = 16 / size;
  const bool fits = x.stride(3) == 1 && x.stride(0) % per16 == 0 && x.stride(1) % per16 == 0 && x.stride(2) % per16 == 0 &&
                    reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && (x.size(1) <= 1 || x.stride(1) * size <= (1 << 24));
  return fits ? x : x.clone(at::MemoryFormat::Contiguous);
}

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Tensor& v0, double scale, double softcap,
                        const OptTensor& slopes, bool causal, const OptTensor& prefix, const OptTensor& q_doc, const OptTensor& k_doc,
                        bool train) {
    const int64_t own = q0.size(3), width = (own + 7) / 8 * 8;
    const Tensor q = ready(q0, width), k = ready(k0, width), v = ready(v0, width);
    auto got = attention_fwd(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc, train);
    if (train) {
      ctx->save_for_backward({q, k, v, got[0], got[1], got[2], slopes.value_or(Tensor()), prefix.value_or(Tensor()),
                              q_doc.value_or(Tensor()), k_doc.value_or(Tensor())});
      ctx->saved_data["scale"] = scale;
      ctx->saved_data["softcap"] = softcap;
      ctx->saved_data["causal"] = causal;
      ctx->saved_data["own"] = own;
    }
    // not a view, which from within a function may not be changed in place
    return own == width ? got[0] : got[0].narrow(3, 0, own).contiguous();
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("attention");
    const auto s = ctx->get_saved_variables();
    const int64_t own = ctx->saved_data["own"].toInt();
    auto got = attention_bwd(ready(grads[0], s[0].size(3)), s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["scale"].toDouble(),
                             ctx->saved_data["softcap"].toDouble(), opt(s[6]), ctx->saved_data["causal"].toBool(), opt(s[7]), opt(s[8]),
                             opt(s[9]));
    variable_list out(11);
    for (int i = 0; i < 3; ++i) out[i] = own == got[i].size(3) ? got[i] : got[i].narrow(3, 0, own);
    return out;
  }
};

}  // namespace

std::vector<Tensor> rms_norm(Tensor x, Tensor weight, OptTensor residual, double eps) {
  check_norm(x, weight, residual);
  capturable({x, weight, residual}, "rms_norm");
  return RmsNorm::apply(x, weight, residual, eps);
}

// {codes, scales} and the sum, if there is a residual.
std::vector<Tensor> rms_norm_fp8(Tensor x, Tensor weight, OptTensor residual, double eps, int64_t group) {
  check_norm(x, weight, residual);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(x.requires_grad() || weight.requires_grad() || (residual.has_value() && residual->requires_grad())),
              "rms_norm_fp8 has no gradient: call it under torch.no_grad()");
  const int64_t D = x.size(-1);
  TORCH_CHECK_VALUE(group == 0 || (group >= 16 && group <= 512 && (group & (group - 1)) == 0 && D % group == 0), "rms_norm_fp8: group ", group,
                    " is not a power of two from 16 to 512 that divides ", D);
  // groups want eight neighbours to a lane: rows that begin off a 16-byte border are copied
  auto placed = [&](const Tensor& t) { return group > 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0 ? t.clone() : t; };
  auto got = rms_norm_fwd(placed(rows(x)), placed(weight.contiguous()), residual.has_value() ? OptTensor(placed(rows(*residual))) : c10::nullopt,
                          eps, group, x.sizes());
  if (x.dim() != 2) {
    auto sizes = x.sizes().vec();
    sizes.back() = got[1].size(1);
    got[1] = got[1].view(sizes);
  }
  return got;
}

std::vector<Tensor> rotary(Tensor q, OptTensor k, Tensor positions, Tensor frequencies, bool interleaved, double amplitude) {
  auto check = [&](const Tensor& x, const char* name) {
    TORCH_CHECK_VALUE(x.dim() == 4, "rotary: ", name, " is [batch, length, heads, width], got ", x.sizes());
    TORCH_CHECK_TYPE(floating(x) && x.scalar_type() == q.scalar_type(), "rotary: q and k are fp32, bf16 or fp16 of one type, got ", name, " ",
                     x.scalar_type());
    TORCH_CHECK_VALUE(x.size(0) == q.size(0) && x.size(1) == q.size(1) && x.size(3) == q.size(3), "rotary: q ", q.sizes(), " and k ", x.sizes(),
                      " do not go together");
  };
  check(q, "q");
  if (k.has_value()) check(*k, "k");
  const int64_t heads = q.size(2) + (k.has_value() ? k->size(2) : 0);
  TORCH_CHECK_VALUE(heads <= 4096 && q.size(3) <= 4096, "rotary: up to 4096 heads of q and k together and widths up to 4096 expected, got ", heads,
                    " of ", q.size(3));
  TORCH_CHECK_TYPE(frequencies.scalar_type() == at::kDouble && (frequencies.dim() == 1 || frequencies.dim() == 2),
                   "rotary: frequencies are fp64 [n] or [axes, n], got ", frequencies.scalar_type(), " ", frequencies.sizes());
  const int64_t P = frequencies.numel();
  TORCH_CHECK_VALUE(P >= 1 && P <= 512 && 2 * P <= q.size(3), "rotary: ", P, " frequencies do not fit heads of ", q.size(3), " (at most 512)");
  TORCH_CHECK_TYPE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, "rotary: positions are int32 or int64, got ",
                   positions.scalar_type());
  TORCH_CHECK(!at::GradMode::is_enabled() || !frequencies.requires_grad(), "rotary: frequencies have no gradient");
  const bool axes = frequencies.dim() == 2;
  const int64_t lead = positions.dim() - axes;
  TORCH_CHECK_VALUE((lead == 1 || lead == 2) && positions.size(lead - 1) == q.size(1) && (lead == 1 || positions.size(0) == q.size(0)) &&
                        (!axes || positions.size(lead) == frequencies.size(0)),
                    "rotary: positions ", positions.sizes(), " do not fit q ", q.sizes(), " and frequencies ", frequencies.sizes());
  for (const Tensor& x : {k.value_or(q), positions, frequencies})
    TORCH_CHECK_VALUE(x.device() == q.device(), "rotary: tensors on ", q.device(), " and ", x.device());
  capturable({q, k}, "rotary");
  if (!axes) positions = positions.unsqueeze(-1);
  if (lead == 1) positions = positions.unsqueeze(0).expand({q.size(0), q.size(1), positions.size(-1)});
  return Rotary::apply(q, k, positions, frequencies.is_contiguous() ? frequencies : frequencies.contiguous(), interleaved, amplitude);
}

Tensor attention(Tensor q, Tensor k, Tensor v, double scale, double softcap, OptTensor slopes, bool causal, OptTensor prefix,
                 OptTensor q_doc, OptTensor k_doc) {
  const bool train = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  capturable({q, k, v}, "attention");
  return Attention::apply(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc, train);
}
