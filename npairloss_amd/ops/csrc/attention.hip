// Attention with capped scores, distance biases and masks: forward and backward
// (gfx950).  The mathematics stands in attention.h.

#include <torch/extension.h>
#include <ATen/DeviceGuard.h>
#include <ATen/hip/HIPContext.h>

#include "attention.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / WAVE;

template <typename T>
__global__ __launch_bounds__(kThreads) void forward_rows_kernel(AttnArgs a, int64_t rows) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / WAVE;
  if (row >= rows) return;
  const int64_t bh = row / a.Lq;
  forward_row<T>(a, bh / a.H, row % a.Lq, bh % a.H);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dq_rows_kernel(AttnArgs a, int64_t rows) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / WAVE;
  if (row >= rows) return;
  const int64_t bh = row / a.Lq;
  dq_row<T>(a, bh / a.H, row % a.Lq, bh % a.H);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dkv_rows_kernel(AttnArgs a, int64_t rows) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / WAVE;
  if (row >= rows) return;
  const int64_t bh = row / a.Lk;
  dkv_row<T>(a, bh / a.Hk, row % a.Lk, bh % a.Hk);
}

// delta[b, h, i] = sum_d dout o: sixteen lanes a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void delta_kernel(AttnArgs a, float* __restrict__ delta, int64_t rows) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 16) + threadIdx.x / 16;
  if (row >= rows) return;  // rows of a wave end together only at a multiple of four: lanes that are left shuffle among themselves
  const int64_t bl = row / a.H;
  const int h = row % a.H, b = bl / a.Lq, i = bl % a.Lq, t = threadIdx.x % 16;
  const T* g = g_row<T>(a, b, i, h);
  const T* o = static_cast<const T*>(a.o) + row * a.D;
  float s = 0.f;
  if (t * 8 < a.D) {
    float x[8], y[8];
    load8(g + t * 8, x);
    load8(o + t * 8, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
  }
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) s += __shfl_xor(s, off, 16);
  if (t == 0) delta[(static_cast<int64_t>(b) * a.H + h) * a.Lq + i] = s;
}

void check_tensor(const torch::Tensor& x, const torch::Tensor& q, const char* name) {
  const int64_t per16 = 16 / x.element_size();
  TORCH_CHECK(x.is_cuda() && x.device() == q.device() && x.dim() == 4 && x.scalar_type() == q.scalar_type(),
              "attention: ", name, " is [batch, length, heads, width] of q's type on its device");
  TORCH_CHECK(x.size(0) == q.size(0) && x.size(3) == q.size(3), "attention: ", name, " does not fit q");
  TORCH_CHECK(x.stride(3) == 1 && x.stride(0) % per16 == 0 && x.stride(1) % per16 == 0 && x.stride(2) % per16 == 0 &&
                  reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "attention: rows of ", name, " begin at 16-byte borders");
}

RowStrides strides_of(const torch::Tensor& x) { return {x.stride(0), x.stride(1), x.stride(2)}; }

const int* ids(const c10::optional<torch::Tensor>& x, const torch::Tensor& q, std::vector<int64_t> shape, const char* name) {
  if (!x.has_value()) return nullptr;
  TORCH_CHECK(x->device() == q.device() && x->scalar_type() == at::kInt && x->is_contiguous() &&
                  x->sizes() == at::IntArrayRef(shape), "attention: ", name, " has another shape, type or device");
  return x->data_ptr<int>();
}

AttnArgs arguments(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, double scale, double softcap,
                   const c10::optional<torch::Tensor>& slopes, bool causal, const c10::optional<torch::Tensor>& prefix,
                   const c10::optional<torch::Tensor>& q_doc, const c10::optional<torch::Tensor>& k_doc) {
  check_tensor(q, q, "q");
  check_tensor(k, q, "k");
  check_tensor(v, q, "v");
  const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), D = q.size(3), Lk = k.size(1), Hk = k.size(2);
  TORCH_CHECK(B > 0 && Lq > 0 && Lk > 0 && H > 0 && Hk > 0 && H % Hk == 0, "attention: empty, or heads that do not divide");
  TORCH_CHECK(D % 8 == 0 && D >= 8 && D <= 128, "attention: widths of 8 to 128 in steps of 8, got ", D);
  TORCH_CHECK(v.size(1) == Lk && v.size(2) == Hk, "attention: k and v differ");
  TORCH_CHECK(std::max(Lq, Lk) < (int64_t{1} << 30) && B * H < (int64_t{1} << 31) / 2 && q_doc.has_value() == k_doc.has_value(),
              "attention: too long, or documents of one side only");
  if (slopes.has_value())
    TORCH_CHECK(slopes->device() == q.device() && slopes->scalar_type() == at::kFloat && slopes->is_contiguous() &&
                    slopes->dim() == 1 && slopes->size(0) == H, "attention: slopes are fp32 [heads]");
  AttnArgs a{};
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
  a.qs = strides_of(q); a.ks = strides_of(k); a.vs = strides_of(v);
  a.B = B; a.Lq = Lq; a.Lk = Lk; a.H = H; a.Hk = Hk; a.D = D;
  a.scale = static_cast<float>(scale);
  a.softcap = static_cast<float>(softcap);
  a.slopes = slopes.has_value() ? slopes->data_ptr<float>() : nullptr;
  a.causal = causal;
  a.prefix = causal ? ids(prefix, q, {B}, "prefix") : nullptr;
  a.q_doc = ids(q_doc, q, {B, Lq}, "documents");
  a.k_doc = ids(k_doc, q, {B, Lk}, "key_documents");
  return a;
}

int blocks_for(int64_t items, int64_t each) {
  const int64_t n = (items + each - 1) / each;
  TORCH_CHECK(n < (int64_t{1} << 31), "attention: too many rows");
  return static_cast<int>(n);
}

}  // namespace

// {o [B, Lq, H, D], lse [B, H, Lq]}
std::vector<torch::Tensor> attention_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, double scale, double softcap,
                                         c10::optional<torch::Tensor> slopes, bool causal,
                                         c10::optional<torch::Tensor> prefix, c10::optional<torch::Tensor> q_doc,
                                         c10::optional<torch::Tensor> k_doc) {
  AttnArgs a = arguments(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc);
  at::DeviceGuard guard(q.device());
  auto o = torch::empty({a.B, a.Lq, a.H, a.D}, q.options());
  auto lse = torch::empty({a.B, a.H, a.Lq}, q.options().dtype(at::kFloat));
  a.o = o.data_ptr();
  a.lse = lse.data_ptr<float>();
  auto stream = at::hip::getCurrentHIPStream();
  const int64_t rows = static_cast<int64_t>(a.B) * a.H * a.Lq;
  DISPATCH_FLOAT(q.scalar_type(), "attention", [&] {
    forward_rows_kernel<T><<<blocks_for(rows, kWaves), kThreads, 0, stream>>>(a, rows);
  });
  HIP_CHECK_LAST();
  return {o, lse};
}

// {dq, dk, dv}, contiguous
std::vector<torch::Tensor> attention_bwd(torch::Tensor dout, torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                         torch::Tensor o, torch::Tensor lse, double scale, double softcap,
                                         c10::optional<torch::Tensor> slopes, bool causal,
                                         c10::optional<torch::Tensor> prefix, c10::optional<torch::Tensor> q_doc,
                                         c10::optional<torch::Tensor> k_doc) {
  AttnArgs a = arguments(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc);
  check_tensor(dout, q, "the gradient");
  TORCH_CHECK(dout.sizes() == q.sizes() && o.sizes() == q.sizes() && o.is_contiguous() && o.scalar_type() == q.scalar_type() &&
                  lse.numel() == static_cast<int64_t>(a.B) * a.H * a.Lq && lse.is_contiguous() && lse.scalar_type() == at::kFloat);
  at::DeviceGuard guard(q.device());
  auto dq = torch::empty({a.B, a.Lq, a.H, a.D}, q.options());
  auto dk = torch::empty({a.B, a.Lk, a.Hk, a.D}, q.options());
  auto dv = torch::empty({a.B, a.Lk, a.Hk, a.D}, q.options());
  auto delta = torch::empty({a.B, a.H, a.Lq}, lse.options());
  a.o = o.data_ptr(); a.lse = lse.data_ptr<float>();
  a.dout = dout.data_ptr(); a.gs = strides_of(dout);
  a.delta = delta.data_ptr<float>();
  a.dq = dq.data_ptr(); a.dk = dk.data_ptr(); a.dv = dv.data_ptr();
  auto stream = at::hip::getCurrentHIPStream();
  const int64_t q_rows = static_cast<int64_t>(a.B) * a.H * a.Lq, k_rows = static_cast<int64_t>(a.B) * a.Hk * a.Lk;
  DISPATCH_FLOAT(q.scalar_type(), "attention", [&] {
    delta_kernel<T><<<blocks_for(q_rows, kThreads / 16), kThreads, 0, stream>>>(a, delta.data_ptr<float>(), q_rows);
    dq_rows_kernel<T><<<blocks_for(q_rows, kWaves), kThreads, 0, stream>>>(a, q_rows);
    dkv_rows_kernel<T><<<blocks_for(k_rows, kWaves), kThreads, 0, stream>>>(a, k_rows);
  });
  HIP_CHECK_LAST();
  return {dq, dk, dv};
}
