// One AdamW step over many tensors, moments in fp32 or in 8 bits (gfx950).
//
//   m' = b1 m + (1 - b1) g        v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// 8 bits: blocks of 256 elements; m and the root of v are held in e4m3 with an
// fp32 scale each, the block's largest magnitude times the fp32 value of 1 / 448.  The
// root, because it halves the range that the exponent has to cover.  Rounding is stochastic: at
// b2 = 0.999 a step moves v by at most a thousandth of itself (but for large
// gradients), far under half a step of any 8-bit float, so rounding to nearest
// would never let it fall.  m goes up or down with the chances that leave its
// mean as it is, the root with those that leave v's mean as it is, and a root
// that is not zero never becomes zero (m might be rounded up to its least value
// over it).  The random bits are a hash of seed, step, tensor, block and
// element: the same call gives the same codes, whatever the launch looks like.
// The arithmetic up to the codes is one IEEE fp32 operation after another, with
// nothing contracted, so that any implementation that takes the same operations
// gets the same codes.  A moment that is not finite becomes a NaN code and is
// left out of its block's scale: only its own element is lost.
//
// Bound by memory: 28 bytes an element with fp32 parameters and moments, 16
// with bf16 parameters, masters and 8-bit moments.  A launch takes up to
// kTensors tensors by value in its arguments (nothing is copied to the device
// first, and a captured launch keeps them), cut into chunks of kChunk elements,
// a workgroup to a chunk.  The count of steps is read on the device, so that a
// captured step counts on; it is raised by a second, tiny kernel behind all the
// workgroups that read it.
//
// 86 million elements in 150 tensors, three launches: 495 us in fp32 (4.9 TB/s), 313 us in
// bf16 with masters and 8-bit moments (4.4 TB/s).

#include <torch/extension.h>
#include <ATen/DeviceGuard.h>
#include <ATen/hip/HIPContext.h>

#include <algorithm>
#include <cmath>
#include <utility>

#include "vec.h"

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;
constexpr int kBlock = 256;    // elements to a scale
constexpr int kTensors = 52;   // of a launch: its arguments stay under 4 KB
constexpr int kMostChunks = 1 << 23;  // of a launch: under 2^32 threads
constexpr int kSteps = 400;    // of a launch that raises counts
constexpr float kFp8Max = 448.f;
constexpr float kInvMax = 1.f / 448.f;
constexpr float kTiny = 1.17549435e-38f;
constexpr float kMinNormal = 0.015625f;  // least normal e4m3

struct Tensor {
  void* p;        // parameter
  const void* g;  // gradient, the parameter's type
  void* m;
  void* v;
  float* master;  // or null: the parameter itself is updated
  float* scale;   // 8 bits: [blocks, 2]
  const int* step;
  int64_t n;
};

struct Args {
  Tensor t[kTensors];
  int first[kTensors + 1];  // chunk at which a tensor begins
  int count;
  uint32_t index0;          // of the first tensor in the caller's list
  uint32_t seed;
  float decay, lr, b1, b2, a1, a2, eps, log_b1, log_b2;  // a = 1 - b; decay = 1 - lr wd
};
static_assert(sizeof(Args) <= 4096, "kernel arguments are at most 4 KB");

struct StepArgs {
  int* step[kSteps];
  int count;
};

DEVINL uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x9E3779B9u;
  x = (x ^ (x >> 15)) * 0xB7E15163u;
  return x ^ (x >> 16);
}

// The coefficients of a step: p' = p * decay - rate * m / (root * inv_c2 + eps)
struct Rates {
  float rate, inv_c2;
  DEVINL Rates(const Args& a, int t) {
    const float ft = static_cast<float>(t);
    rate = a.lr / -expm1f(ft * a.log_b1);
    inv_c2 = 1.f / sqrtf(-expm1f(ft * a.log_b2));
  }
};

DEVINL float updated(float p, float m, float root, const Args& a, const Rates& r) {
  return p * a.decay - r.rate * (m / (root * r.inv_c2 + a.eps));
}

// `low` is what is added so that numbers below the least normal one round on its grid.
DEVINL float grid_offset(float a) { return a < kMinNormal ? kMinNormal : 0.f; }

// |x| (at most 448) up or down to e4m3, up with chance (distance / step); `dither`
// is 20 random bits.
DEVINL float dithered(float x, uint32_t dither) {
#pragma clang fp contract(off)
  float a = fminf(fabsf(x), kFp8Max);
  const float low = grid_offset(a);
  a = __uint_as_float((__float_as_uint(a + low) + dither) & ~0xFFFFFu) - low;
  return copysignf(fminf(a, kFp8Max), x);
}

// A root in [0, 448] up or down to e4m3, so that its square is right in the mean.
DEVINL float dithered_root(float a, float chance) {
#pragma clang fp contract(off)
  a = fminf(a, kFp8Max);
  const float low = grid_offset(a);
  const uint32_t cut = __float_as_uint(a + low) & ~0xFFFFFu;
  const float down = __uint_as_float(cut) - low;
  const float up = __uint_as_float(cut + 0x100000u) - low;
  const bool rise = chance * ((up - down) * (up + down)) < (a - down) * (a + down);
  const float r = fminf(rise ? up : down, kFp8Max);
  return (a > 0.f && r == 0.f) ? 0.001953125f : r;
}

template <typename T>
DEVINL void load_some(const T* p, int n, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < n ? to_f(p[e]) : 0.f;
}

template <typename T>
DEVINL void store_some(T* p, int n, const float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) p[e] = from_f<T>(v[e]);
}

template <typename T>
DEVINL void load_n(const T* p, int n, bool wide, float (&v)[8]) {
  if (wide) load8(p, v); else load_some(p, n, v);
}

template <typename T>
DEVINL void store_n(T* p, int n, bool wide, const float (&v)[8]) {
  if (wide) store8(p, v); else store_some(p, n, v);
}

DEVINL int find_tensor(const Args& a, int chunk) {  // the last that begins at or before it
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

DEVINL bool wide_ready(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T, bool EIGHT>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Args a) {
  const int which = find_tensor(a, blockIdx.x);
  const Tensor t = a.t[which];
  const int64_t begin = static_cast<int64_t>(blockIdx.x - a.first[which]) * kChunk;
  const int step = *t.step + 1;
  const Rates rates(a, step);
  T* p = static_cast<T*>(t.p);
  const T* g = static_cast<const T*>(t.g);
  const bool ready = wide_ready(t.p) && wide_ready(t.master) && wide_ready(t.m) && wide_ready(t.v);
  const bool g_ready = wide_ready(t.g);  // a view into a gradient bucket may begin anywhere
  uint32_t key0 = 0;
  if (EIGHT) key0 = mix(a.seed + static_cast<uint32_t>(step) * 0x9E3779B9u) ^ ((a.index0 + which) * 0xB7E15163u);
  if (EIGHT) key0 = mix(key0);

  for (int64_t at = begin + threadIdx.x * 8; at < begin + kChunk; at += kThreads * 8) {
    if (!EIGHT && at >= t.n) break;
    // in 8 bits all lanes of a block's 32 stay for its maximum
    const int n = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(8), t.n - at)));
    const bool wide = ready && n == 8;
    float w[8], gv[8], m[8], v[8];
    load_n(g + at, n, g_ready && n == 8, gv);
    if (t.master != nullptr) load_n(t.master + at, n, wide, w); else load_n(p + at, n, wide, w);
    if (!EIGHT) {
      float* mp = static_cast<float*>(t.m);
      float* vp = static_cast<float*>(t.v);
      load_n(mp + at, n, wide, m);
      load_n(vp + at, n, wide, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] = m[e] * a.b1 + gv[e] * a.a1;
        v[e] = v[e] * a.b2 + gv[e] * gv[e] * a.a2;
        w[e] = updated(w[e], m[e], sqrtf(v[e]), a, rates);
      }
      store_n(mp + at, n, wide, m);
      store_n(vp + at, n, wide, v);
    } else {
#pragma clang fp contract(off)
      uint8_t* mc = static_cast<uint8_t*>(t.m);
      uint8_t* vc = static_cast<uint8_t*>(t.v);
      const int64_t block = at / kBlock;
      const bool any = block * kBlock < t.n;
      const float2 old = any ? *reinterpret_cast<const float2*>(t.scale + block * 2) : make_float2(0.f, 0.f);
      uint32_t mw[2] = {0, 0}, vw[2] = {0, 0};
      if (wide) {
        *reinterpret_cast<uint2*>(mw) = *reinterpret_cast<const uint2*>(mc + at);
        *reinterpret_cast<uint2*>(vw) = *reinterpret_cast<const uint2*>(vc + at);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) {
            mw[e / 4] |= static_cast<uint32_t>(mc[at + e]) << (8 * (e % 4));
            vw[e / 4] |= static_cast<uint32_t>(vc[at + e]) << (8 * (e % 4));
          }
      }
      float top_m = 0.f, top_v = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float cm = e % 4 == 0   ? __builtin_amdgcn_cvt_f32_fp8(mw[e / 4], 0)
                         : e % 4 == 1 ? __builtin_amdgcn_cvt_f32_fp8(mw[e / 4], 1)
                         : e % 4 == 2 ? __builtin_amdgcn_cvt_f32_fp8(mw[e / 4], 2)
                                      : __builtin_amdgcn_cvt_f32_fp8(mw[e / 4], 3);
        const float cv = e % 4 == 0   ? __builtin_amdgcn_cvt_f32_fp8(vw[e / 4], 0)
                         : e % 4 == 1 ? __builtin_amdgcn_cvt_f32_fp8(vw[e / 4], 1)
                         : e % 4 == 2 ? __builtin_amdgcn_cvt_f32_fp8(vw[e / 4], 2)
                                      : __builtin_amdgcn_cvt_f32_fp8(vw[e / 4], 3);
        m[e] = cm * old.x;
        v[e] = cv * old.y;
        v[e] = v[e] * v[e];
        m[e] = m[e] * a.b1 + gv[e] * a.a1;
        v[e] = v[e] * a.b2 + (gv[e] * gv[e]) * a.a2;
        v[e] = sqrtf(v[e]);
        if (fabsf(m[e]) <= FLT_MAX) top_m = fmaxf(top_m, fabsf(m[e]));
        if (v[e] <= FLT_MAX) top_v = fmaxf(top_v, v[e]);
      }
#pragma unroll
      for (int off = kBlock / 16; off > 0; off >>= 1) {
        top_m = fmaxf(top_m, __shfl_xor(top_m, off, WAVE));
        top_v = fmaxf(top_v, __shfl_xor(top_v, off, WAVE));
      }
      const float sm = fmaxf(top_m * kInvMax, kTiny), sv = fmaxf(top_v * kInvMax, kTiny);
      const float im = 1.f / sm, iv = 1.f / sv;
      const uint32_t key = mix(key0 ^ static_cast<uint32_t>(block));
      const uint32_t inside = static_cast<uint32_t>(at % kBlock);
      float rm[8], rv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t bits = mix(key + (inside + e) * 0x9E3779B9u);
        rm[e] = fabsf(m[e]) <= FLT_MAX ? dithered(m[e] * im, ((bits & 0xFFFFu) << 4) | 8u) : __builtin_nanf("");
        const float chance = (static_cast<float>(bits >> 16) + 0.5f) * 1.52587890625e-5f;
        rv[e] = v[e] <= FLT_MAX ? dithered_root(v[e] * iv, chance) : __builtin_nanf("");
        w[e] = updated(w[e], m[e], v[e], a, rates);
      }
      mw[0] = pack_fp8(rm[0], rm[1], rm[2], rm[3]);
      mw[1] = pack_fp8(rm[4], rm[5], rm[6], rm[7]);
      vw[0] = pack_fp8(rv[0], rv[1], rv[2], rv[3]);
      vw[1] = pack_fp8(rv[4], rv[5], rv[6], rv[7]);
      if (wide) {
        *reinterpret_cast<uint2*>(mc + at) = *reinterpret_cast<const uint2*>(mw);
        *reinterpret_cast<uint2*>(vc + at) = *reinterpret_cast<const uint2*>(vw);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) {
            mc[at + e] = (mw[e / 4] >> (8 * (e % 4))) & 0xFF;
            vc[at + e] = (vw[e / 4] >> (8 * (e % 4))) & 0xFF;
          }
      }
      if (any && inside == 0) *reinterpret_cast<float2*>(t.scale + block * 2) = make_float2(sm, sv);
    }
    if (t.master != nullptr) store_n(t.master + at, n, wide, w);
    store_n(p + at, n, wide, w);
  }
}

__global__ __launch_bounds__(kSteps) void raise_steps_kernel(StepArgs a) {
  if (static_cast<int>(threadIdx.x) < a.count) ++*a.step[threadIdx.x];
}

}  // namespace

// One step in place.  The lists go together; `masters` and `scales` are empty or as
// long.  Checked here and not in Python, where a hundred tensors take longer than
// their step.
void adamw_update(std::vector<torch::Tensor> params, std::vector<torch::Tensor> grads,
                  std::vector<torch::Tensor> ms, std::vector<torch::Tensor> vs,
                  std::vector<torch::Tensor> steps, std::vector<torch::Tensor> masters,
                  std::vector<torch::Tensor> scales, double lr, double b1, double b2, double eps,
                  double weight_decay, int64_t seed) {
  const size_t count = params.size();
  if (count == 0) return;
  const bool eight = !scales.empty();
  TORCH_CHECK_VALUE(grads.size() == count && ms.size() == count && vs.size() == count && steps.size() == count &&
                        (masters.empty() || masters.size() == count) && (!eight || scales.size() == count),
                    "adamw_step: lists of different lengths");
  const auto device = params[0].device();
  const auto type = params[0].scalar_type();
  TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, "adamw_step: fp32, bf16 or fp16 parameters expected, got ", type);
  const auto state = eight ? at::kFloat8_e4m3fn : at::kFloat;
  // whether elements of two tensors of one shape lie in memory in the same order
  auto like = [](const torch::Tensor& x, const torch::Tensor& y) {
    for (int64_t d = 0; d < y.dim(); ++d)
      if (y.size(d) > 1 && x.stride(d) != y.stride(d)) return false;
    return true;
  };
  for (size_t i = 0; i < count; ++i) {
    const auto& p = params[i];
    const int64_t n = p.numel();
    auto fits = [&](const torch::Tensor& x, at::ScalarType want) {
      return x.layout() == at::kStrided && x.device() == device && x.scalar_type() == want && x.sizes() == p.sizes();
    };
    TORCH_CHECK_VALUE(fits(p, type) && p.is_cuda(), "adamw_step: parameter ", i, " is ", p.scalar_type(), " on ", p.device(),
                      ", the first ", type, " on ", device);
    TORCH_CHECK_VALUE(n == 0 || p.is_non_overlapping_and_dense(), "adamw_step: parameter ", i, " does not fill a stretch of memory");
    TORCH_CHECK_VALUE(fits(grads[i], type), "adamw_step: gradient ", i, " does not fit its parameter");
    TORCH_CHECK_VALUE(fits(ms[i], state) && like(ms[i], p) && fits(vs[i], state) && like(vs[i], p), "adamw_step: moments ", i,
                      " are not laid out as their parameter in ", state);
    TORCH_CHECK_VALUE(masters.empty() || (fits(masters[i], at::kFloat) && like(masters[i], p)), "adamw_step: master ", i,
                      " is not laid out as its parameter in fp32");
    TORCH_CHECK_VALUE(steps[i].device() == device && steps[i].scalar_type() == at::kInt && steps[i].numel() == 1, "adamw_step: step ", i,
                      " is one int32 on ", device);
    TORCH_CHECK_VALUE(!eight || (scales[i].device() == device && scales[i].scalar_type() == at::kFloat && scales[i].is_contiguous() &&
                                 scales[i].dim() == 2 && scales[i].size(0) == (n + kBlock - 1) / kBlock && scales[i].size(1) == 2 &&
                                 reinterpret_cast<uintptr_t>(scales[i].data_ptr()) % 8 == 0),
                      "adamw_step: scales ", i, " are not fp32 [blocks of ", kBlock, ", 2]");
    TORCH_CHECK_VALUE(n <= int64_t{kMostChunks} * kChunk, "adamw_step: parameter ", i, " is too large");
  }
  const auto lists = {&params, &ms, &vs, &steps, &masters, &scales};
  std::vector<std::pair<uintptr_t, uintptr_t>> written;  // what comes twice would be updated by two workgroups at once
  for (const auto* list : lists)
    for (const auto& x : *list)
      if (x.numel() > 0) {
        const auto begin = reinterpret_cast<uintptr_t>(x.data_ptr());
        written.emplace_back(begin, begin + x.numel() * x.element_size());
      }
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    TORCH_CHECK(written[i - 1].second <= written[i].first, "adamw_step: a tensor comes twice, or overlaps another");
  for (const auto* list : lists)  // a graph that has saved one of them learns of the change
    for (const auto& x : *list) x.unsafeGetTensorImpl()->bump_version();
  at::DeviceGuard guard(device);
  for (size_t i = 0; i < count; ++i)  // gradients in another order of dimensions are brought into the parameter's
    if (!like(grads[i], params[i])) grads[i] = torch::empty_like(params[i]).copy_(grads[i]);
  auto stream = at::hip::getCurrentHIPStream();
  Args a;
  a.seed = static_cast<uint32_t>(seed);
  a.decay = static_cast<float>(1.0 - lr * weight_decay);
  a.lr = static_cast<float>(lr);
  a.b1 = static_cast<float>(b1);
  a.b2 = static_cast<float>(b2);
  a.a1 = static_cast<float>(1.0 - b1);
  a.a2 = static_cast<float>(1.0 - b2);
  a.eps = static_cast<float>(eps);
  a.log_b1 = static_cast<float>(std::log(b1));
  a.log_b2 = static_cast<float>(std::log(b2));
  int64_t chunks = 0;
  auto flush = [&](size_t next) {
    if (chunks > 0) {
      DISPATCH_FLOAT(type, "adamw_step", [&] {
        if (eight) adamw_kernel<T, true><<<static_cast<int>(chunks), kThreads, 0, stream>>>(a);
        else adamw_kernel<T, false><<<static_cast<int>(chunks), kThreads, 0, stream>>>(a);
      });
      HIP_CHECK_LAST();
    }
    a.count = 0;
    chunks = 0;
    a.index0 = static_cast<uint32_t>(next);
  };
  a.count = 0;
  a.index0 = 0;
  for (size_t i = 0; i < count; ++i) {
    const int64_t n = params[i].numel(), more = (n + kChunk - 1) / kChunk;
    if (a.count == kTensors || (a.count > 0 && chunks + more > kMostChunks)) flush(i);
    a.t[a.count] = Tensor{params[i].data_ptr(), grads[i].data_ptr(), ms[i].data_ptr(), vs[i].data_ptr(),
                          masters.empty() ? nullptr : masters[i].data_ptr<float>(),
                          eight ? scales[i].data_ptr<float>() : nullptr, steps[i].data_ptr<int>(), n};
    a.first[a.count] = static_cast<int>(chunks);
    chunks += more;
    a.first[++a.count] = static_cast<int>(chunks);
  }
  flush(count);
  for (size_t i = 0; i < count; i += kSteps) {
    StepArgs s;
    s.count = static_cast<int>(std::min<size_t>(kSteps, count - i));
    for (int j = 0; j < s.count; ++j) s.step[j] = steps[i + j].data_ptr<int>();
    raise_steps_kernel<<<1, kSteps, 0, stream>>>(s);
    HIP_CHECK_LAST();
  }
}
