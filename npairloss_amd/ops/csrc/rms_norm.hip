// Root-mean-square norm over rows, with the residual's addition in front and
// an output in the input's type or in e4m3 with scales (gfx950).
//
//   s = x + r            rounded once to the type the caller keeps it in
//   y = s * inv * w      inv = rsqrt(mean(s^2) + eps)
//   e4m3: code = y / scale, scale = max|y| / 448 over a row or a group of it
//
//   g = w * dy
//   ds_total = ds + inv * (g - s * inv^2 * mean(g * s))
//   dw       = sum over rows of dy * s * inv
//
// All of it is bound by memory: a row is read once into registers, reduced,
// and written once.  A row belongs to 64 threads up to 2048 columns (four rows
// to a workgroup, no barrier), to 256 up to 4096 (e4m3: 8192), to 1024 up to 16384,
// so that it fits in at most 32 registers a thread.  Rows whose width or address is
// not a multiple of eight elements take the same kernels with one element to
// an access, neighbouring lanes on neighbouring elements.
//
// 12608 rows of 768 bf16 with a residual: 14.7 us forward (5.3 TB/s), 20.9 backward with the
// weight's sums (3.7 TB/s: a workgroup walks over rows to keep the weight's gradient in registers, and each
// waits for its row); 16384 rows of 8192 bf16 with a residual to e4m3 in groups of 128: 194 us
// (4.8 TB/s); one row of 4096: 4 us, a launch.

#include <torch/extension.h>
#include <ATen/DeviceGuard.h>
#include <ATen/hip/HIPContext.h>
#include <c10/util/accumulate.h>

#include "vec.h"

namespace {

constexpr float kFp8Max = 448.f;
constexpr float kTiny = 1.17549435e-38f;  // least normal fp32: the least scale

// Where element e of a thread's chunk k lies in its row.
template <bool VEC, int TPR>
DEVINL int column(int t, int k, int e) {
  return VEC ? (t + k * TPR) * 8 + e : t + (k * 8 + e) * TPR;
}

template <typename T, bool VEC, int TPR>
DEVINL void load_row(const T* __restrict__ row, int t, int k, int D, float (&v)[8]) {
  if (VEC) {
    if (column<VEC, TPR>(t, k, 0) < D) {
      load8(row + column<VEC, TPR>(t, k, 0), v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = column<VEC, TPR>(t, k, e);
      v[e] = c < D ? to_f(row[c]) : 0.f;
    }
  }
}

template <typename T, bool VEC, int TPR>
DEVINL void store_row(T* __restrict__ row, int t, int k, int D, const float (&v)[8]) {
  if (VEC) {
    if (column<VEC, TPR>(t, k, 0) < D) store8(row + column<VEC, TPR>(t, k, 0), v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = column<VEC, TPR>(t, k, e);
      if (c < D) row[c] = from_f<T>(v[e]);
    }
  }
}

template <typename T, bool VEC, int TPR>
DEVINL void load_weight(const void* w, bool w_f32, int t, int k, int D, float (&v)[8]) {
  if (w_f32)
    load_row<float, VEC, TPR>(static_cast<const float*>(w), t, k, D, v);
  else
    load_row<T, VEC, TPR>(static_cast<const T*>(w), t, k, D, v);
}

struct AddOp { DEVINL float operator()(float a, float b) const { return a + b; } };
struct MaxOp { DEVINL float operator()(float a, float b) const { return max_or_nan(a, b); } };

// Over the TPR threads of a row.  `scratch`: one float a wave.
template <int TPR, typename Op>
DEVINL float row_reduce(float v, Op op, float* scratch) {
#pragma unroll
  for (int off = WAVE / 2; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off, WAVE));
  if (TPR == WAVE) return v;
  constexpr int kWaves = TPR / WAVE;
  __syncthreads();  // the last call's values have been read
  if (threadIdx.x % WAVE == 0) scratch[threadIdx.x / WAVE] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) v = op(v, scratch[i]);
  return v;
}

template <typename T, bool VEC, int TPR, int NCH, bool FP8>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_fwd_kernel(
    const T* __restrict__ x, const T* __restrict__ residual, const void* __restrict__ w,
    bool w_f32, float eps, int64_t N, int D, int group, T* __restrict__ sum,
    T* __restrict__ y, float* __restrict__ inv_out, uint8_t* __restrict__ codes,
    float* __restrict__ scales) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  __shared__ float scratch[kThreads / WAVE];
  const int t = threadIdx.x % TPR;
  const int64_t row = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * (kThreads / TPR) + threadIdx.x / TPR;
  if (row >= N) return;  // whole waves; with TPR > 64 there is one row a block
  const int64_t at = row * D;

  float v[NCH][8];
#pragma unroll
  for (int k = 0; k < NCH; ++k) load_row<T, VEC, TPR>(x + at, t, k, D, v[k]);
  if (residual != nullptr) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      float r[8];
      load_row<T, VEC, TPR>(residual + at, t, k, D, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = to_f(from_f<T>(v[k][e] + r[e]));
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) store_row<T, VEC, TPR>(sum + at, t, k, D, v[k]);
  }

  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += v[k][e] * v[k][e];
  ss = row_reduce<TPR>(ss, AddOp(), scratch);
  const float inv = 1.f / sqrtf(ss / static_cast<float>(D) + eps);
  if (inv_out != nullptr && t == 0) inv_out[row] = inv;

#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    float wv[8];
    load_weight<T, VEC, TPR>(w, w_f32, t, k, D, wv);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = v[k][e] * inv * wv[e];
  }
  if (!FP8) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) store_row<T, VEC, TPR>(y + at, t, k, D, v[k]);
    return;
  }

  float top[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    top[k] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top[k] = max_or_nan(fabsf(v[k][e]), top[k]);
  }
  if (group == 0) {  // one scale a row
    float m = top[0];
#pragma unroll
    for (int k = 1; k < NCH; ++k) m = max_or_nan(top[k], m);
    m = row_reduce<TPR>(m, MaxOp(), scratch);
#pragma unroll
    for (int k = 0; k < NCH; ++k) top[k] = m;
  } else {  // group / 8 neighbouring lanes hold a group
    for (int off = group / 16; off > 0; off >>= 1)
#pragma unroll
      for (int k = 0; k < NCH; ++k) top[k] = max_or_nan(top[k], __shfl_xor(top[k], off, WAVE));
  }
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    float scale = top[k] / kFp8Max;
    scale = scale < kTiny ? kTiny : scale;  // keeps NaN
    const float mul = 1.f / scale;
    const int c = column<VEC, TPR>(t, k, 0);
    if (group == 0) {
      if (t == 0 && k == 0) scales[row] = scale;
    } else if (c < D && c % group == 0) {
      scales[row * (D / group) + c / group] = scale;
    }
    if (VEC) {
      if (c < D) {
        uint2 out;
        out.x = pack_fp8(v[k][0] * mul, v[k][1] * mul, v[k][2] * mul, v[k][3] * mul);
        out.y = pack_fp8(v[k][4] * mul, v[k][5] * mul, v[k][6] * mul, v[k][7] * mul);
        *reinterpret_cast<uint2*>(codes + at + c) = out;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int ce = column<VEC, TPR>(t, k, e);
        if (ce < D) codes[at + ce] = pack_fp8(v[k][e] * mul, 0.f, 0.f, 0.f) & 0xFF;
      }
    }
  }
}

// Each workgroup takes every grid-th group of rows and keeps the weight's
// gradient of its columns in registers; `part` gets one row of sums from each.
template <typename T, bool VEC, int TPR, int NCH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ dsum, const T* __restrict__ s,
    const void* __restrict__ w, bool w_f32, const float* __restrict__ inv_in, int64_t N, int D,
    T* __restrict__ dx, float* __restrict__ part) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  constexpr int kRows = kThreads / TPR;
  __shared__ float scratch[kThreads / WAVE];
  __shared__ float join[kRows > 1 ? (kRows - 1) * NCH * TPR * 8 : 1];
  const int t = threadIdx.x % TPR;
  const int sub = threadIdx.x / TPR;

  float wv[NCH][8], acc[NCH][8];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    load_weight<T, VEC, TPR>(w, w_f32, t, k, D, wv[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[k][e] = 0.f;
  }
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub; row < N;
       row += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t at = row * D;
    const float inv = inv_in[row];
    float sv[NCH][8], g[NCH][8], dot = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      load_row<T, VEC, TPR>(s + at, t, k, D, sv[k]);
      load_row<T, VEC, TPR>(dy + at, t, k, D, g[k]);
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sv[k][e] *= inv;  // the normalised row
        acc[k][e] += g[k][e] * sv[k][e];
        g[k][e] *= wv[k][e];
        dot += g[k][e] * sv[k][e];
      }
    dot = row_reduce<TPR>(dot, AddOp(), scratch) / static_cast<float>(D);
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      float o[8];
      if (dsum != nullptr) {
        load_row<T, VEC, TPR>(dsum + at, t, k, D, o);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += inv * (g[k][e] - sv[k][e] * dot);
      store_row<T, VEC, TPR>(dx + at, t, k, D, o);
    }
  }
  if (kRows > 1) {
    if (sub > 0) {
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) join[((sub - 1) * NCH * 8 + k * 8 + e) * TPR + t] = acc[k][e];
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int r = 0; r < kRows - 1; ++r)
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[k][e] += join[(r * NCH * 8 + k * 8 + e) * TPR + t];
  }
#pragma unroll
  for (int k = 0; k < NCH; ++k)
    store_row<float, VEC, TPR>(part + static_cast<int64_t>(blockIdx.x) * D, t, k, D, acc[k]);
}

// Column sums of `part` [G, D] in a fixed order: 32 columns and 32 rows at once.
template <typename W>
__global__ __launch_bounds__(1024) void rms_dweight_kernel(const float* __restrict__ part, int G,
                                                           int D, W* __restrict__ dw) {
  __shared__ float join[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x % 32;
  const int r0 = threadIdx.x / 32;
  float a = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int r = r0; r < G; r += 32) a += part[static_cast<int64_t>(r) * D + c];
  }
  join[r0][threadIdx.x % 32] = a;
  __syncthreads();
  if (r0 != 0 || c >= D) return;
  for (int r = 1; r < 32; ++r) a += join[r][threadIdx.x];
  dw[c] = from_f<W>(a);
}

bool aligned(const void* p) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Calls `fn` with the threads and chunks of a row as constants.  Few threads need no barrier,
// many have a row in flight sooner: bf16, us: 12608 rows of 768 in 64 threads 8.5, in 256 12.7;
// 8192 of 2048 14.7 : 14.1 and with the gradient 39.6 : 41.1; 4096 of 8192 in 256 25.5, in 1024
// 23.9, with the gradient 82 : 68, but in e4m3 29 : 32 (its row is looked at twice more).
template <bool FP8, typename Fn>
void with_width(int64_t D, Fn fn) {
  using std::integral_constant;
  if (D <= 512) fn(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (D <= 1024) fn(integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (D <= 2048) fn(integral_constant<int, 64>(), integral_constant<int, 4>());
  else if (D <= 4096) fn(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (D <= 8192) fn(integral_constant<int, FP8 ? 256 : 1024>(), integral_constant<int, FP8 ? 4 : 1>());
  else fn(integral_constant<int, 1024>(), integral_constant<int, 2>());
}

void check_rows(const torch::Tensor& x, const torch::Tensor& w) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), "rms_norm: contiguous rows expected");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= 16384, "rms_norm: 1 to 16384 columns expected, got ", x.size(1));
  TORCH_CHECK(w.device() == x.device() && w.dim() == 1 && w.size(0) == x.size(1) && w.is_contiguous() &&
                  (w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat),
              "rms_norm: the weight is one row of the input's type or fp32, on its device");
  TORCH_CHECK(x.size(0) < (int64_t{1} << 31), "rms_norm: too many rows");
}

void check_like(const torch::Tensor& x, const c10::optional<torch::Tensor>& r) {
  if (r.has_value())
    TORCH_CHECK(r->device() == x.device() && r->sizes() == x.sizes() && r->is_contiguous() &&
                    r->scalar_type() == x.scalar_type(),
                "rms_norm: rows of the same shape, type and device expected");
}

}  // namespace

// {y or codes, scales (e4m3) or inv, sum (if there is a residual)}, y, codes and sum in
// `shape`.  `group` < 0: y in x's type; 0: e4m3 with a scale a row; > 0: with a scale for
// every group.
std::vector<torch::Tensor> rms_norm_fwd(torch::Tensor x, torch::Tensor weight,
                                        c10::optional<torch::Tensor> residual, double eps,
                                        int64_t group, at::IntArrayRef shape) {
  check_rows(x, weight);
  check_like(x, residual);
  TORCH_CHECK(c10::multiply_integers(shape) == x.numel(), "rms_norm: rows and shape differ");
  const int64_t N = x.size(0), D = x.size(1);
  const bool fp8 = group >= 0;
  TORCH_CHECK(group <= 0 || ((group & (group - 1)) == 0 && group >= 16 && group <= 512 && D % group == 0),
              "rms_norm: a group is a power of two from 16 to 512 that divides the row");
  at::DeviceGuard guard(x.device());
  auto y = torch::empty(shape, fp8 ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
  auto second = fp8 ? torch::empty({N, group > 0 ? D / group : 1}, x.options().dtype(at::kFloat))
                    : torch::empty({N}, x.options().dtype(at::kFloat));
  torch::Tensor sum = residual.has_value() ? torch::empty(shape, x.options()) : torch::Tensor();
  std::vector<torch::Tensor> out{y, second};
  if (residual.has_value()) out.push_back(sum);
  if (N == 0) return out;
  const void* r = residual.has_value() ? residual->data_ptr() : nullptr;
  const bool vec = D % 8 == 0 && aligned(x.data_ptr()) && aligned(weight.data_ptr()) && aligned(r);
  TORCH_CHECK(vec || group <= 0, "rms_norm: groups need rows aligned to 16 bytes");
  const bool w_f32 = weight.scalar_type() == at::kFloat;
  auto stream = at::hip::getCurrentHIPStream();
  DISPATCH_FLOAT(x.scalar_type(), "rms_norm", [&] {
    auto run = [&](auto eight) {
      constexpr bool FP8 = decltype(eight)::value;
      with_width<FP8>(D, [&](auto tpr, auto nch) {
        constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value;
        constexpr int kThreads = TPR > 256 ? TPR : 256;
        const int64_t blocks = (N + kThreads / TPR - 1) / (kThreads / TPR), across = std::min<int64_t>(blocks, (int64_t{1} << 31) / kThreads);
        const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>((blocks + across - 1) / across));
        auto launch = [&](auto kernel) {
          kernel<<<grid, kThreads, 0, stream>>>(
              static_cast<const T*>(x.data_ptr()), static_cast<const T*>(r), weight.data_ptr(), w_f32,
              static_cast<float>(eps), N, static_cast<int>(D), static_cast<int>(FP8 ? group : 0),
              residual.has_value() ? static_cast<T*>(sum.data_ptr()) : nullptr,
              FP8 ? nullptr : static_cast<T*>(y.data_ptr()), FP8 ? nullptr : second.data_ptr<float>(),
              FP8 ? static_cast<uint8_t*>(y.data_ptr()) : nullptr, FP8 ? second.data_ptr<float>() : nullptr);
        };
        if (vec) launch(rms_fwd_kernel<T, true, TPR, NCH, FP8>);
        else launch(rms_fwd_kernel<T, false, TPR, NCH, FP8>);
      });
    };
    if (fp8) run(std::true_type());
    else run(std::false_type());
  });
  HIP_CHECK_LAST();
  return out;
}

// {gradient of the sum (and so of both its terms), gradient of the weight}.
std::vector<torch::Tensor> rms_norm_bwd(torch::Tensor dy, c10::optional<torch::Tensor> dsum,
                                        torch::Tensor s, torch::Tensor weight, torch::Tensor inv) {
  check_rows(s, weight);
  check_like(s, dy);
  check_like(s, dsum);
  const int64_t N = s.size(0), D = s.size(1);
  TORCH_CHECK(inv.device() == s.device() && inv.scalar_type() == at::kFloat && inv.numel() == N && inv.is_contiguous());
  at::DeviceGuard guard(s.device());
  auto dx = torch::empty_like(s);
  auto dw = torch::empty_like(weight);
  if (N == 0) return {dx, dw.zero_()};
  const void* d = dsum.has_value() ? dsum->data_ptr() : nullptr;
  const bool vec = D % 8 == 0 && aligned(s.data_ptr()) && aligned(dy.data_ptr()) &&
                   aligned(weight.data_ptr()) && aligned(d);
  const bool w_f32 = weight.scalar_type() == at::kFloat;
  auto stream = at::hip::getCurrentHIPStream();
  DISPATCH_FLOAT(s.scalar_type(), "rms_norm", [&] {
    with_width<false>(D, [&](auto tpr, auto nch) {
      constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value;
      constexpr int kThreads = TPR > 256 ? TPR : 256;
      constexpr int kRows = kThreads / TPR;
      // Two workgroups a CU of 256 threads, one of 1024: each writes a row of sums, which are
      // read again.  Four where 16-bit rows of few registers leave each three rows and more:
      // bf16, two against four, us: 12608 rows of 768 23.5 : 19.3, 32768 of 512 29 : 23, 8192
      // of 4096 79 : 58, but 8192 of 2048 27.5 : 30.9 and 12608 of 768 fp32 27.9 : 29.8.
      const int64_t steps = (N + kRows - 1) / kRows;
      const bool four = sizeof(T) == 2 && NCH <= 2 && steps >= 3 * 1024;
      const int64_t grid = std::min<int64_t>(steps, TPR > 256 ? 256 : four ? 1024 : 512);
      auto part = torch::empty({grid, D}, s.options().dtype(at::kFloat));
      auto launch = [&](auto kernel) {
        kernel<<<grid, kThreads, 0, stream>>>(
            static_cast<const T*>(dy.data_ptr()), static_cast<const T*>(d),
            static_cast<const T*>(s.data_ptr()), weight.data_ptr(), w_f32, inv.data_ptr<float>(), N,
            static_cast<int>(D), static_cast<T*>(dx.data_ptr()), part.data_ptr<float>());
      };
      if (vec) launch(rms_bwd_kernel<T, true, TPR, NCH>);
      else launch(rms_bwd_kernel<T, false, TPR, NCH>);
      const int blocks = static_cast<int>((D + 31) / 32);
      if (w_f32)
        rms_dweight_kernel<float><<<blocks, 1024, 0, stream>>>(part.data_ptr<float>(), grid, D, dw.data_ptr<float>());
      else
        rms_dweight_kernel<T><<<blocks, 1024, 0, stream>>>(part.data_ptr<float>(), grid, D, static_cast<T*>(dw.data_ptr()));
    });
  });
  HIP_CHECK_LAST();
  return {dx, dw};
}
