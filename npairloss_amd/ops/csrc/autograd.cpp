// The transformer operators as differentiable calls on GPU tensors.  Recorded here
// and not in Python: a pass over a few MB takes the GPU some 15 us, and a Python
// function forward and backward twice that and more.

#include <torch/extension.h>

#include <vector>

std::vector<torch::Tensor> rms_norm_fwd(torch::Tensor x, torch::Tensor weight, c10::optional<torch::Tensor> residual,
                                        double eps, int64_t group);
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

Tensor rows(const Tensor& x) { return x.reshape({-1, x.size(-1)}).contiguous(); }

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
    const Tensor w = weight.contiguous();
    auto got = rms_norm_fwd(rows(x), w, residual.has_value() ? OptTensor(rows(*residual)) : c10::nullopt, eps, -1);
    variable_list out{got[0].view(x.sizes())};
    if (residual.has_value()) out.push_back(got[2].view(x.sizes()));
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
    const Tensor dx = got[0].view(saved[0].sizes());
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
  if (x.size(3) != width) return at::constant_pad_nd(x, {0, width - x.size(3)});
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
    // saved as it lies, given out as a view of its own, so that the node does not hold itself
    return own == width ? got[0].view(got[0].sizes()) : got[0].narrow(3, 0, own);
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
  return RmsNorm::apply(x, weight, residual, eps);
}

std::vector<Tensor> rotary(Tensor q, OptTensor k, Tensor positions, Tensor frequencies, bool interleaved, double amplitude) {
  return Rotary::apply(q, k, positions, frequencies, interleaved, amplitude);
}

Tensor attention(Tensor q, Tensor k, Tensor v, double scale, double softcap, OptTensor slopes, bool causal, OptTensor prefix,
                 OptTensor q_doc, OptTensor k_doc) {
  const bool train = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  return Attention::apply(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc, train);
}
