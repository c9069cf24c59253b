// Rotary positions for queries and keys in one launch (gfx950).
//
// Pair i of a head is turned by the angle p f_i: (a, b) -> (a c - b z, a z + b c)
// with c, z = amplitude * cos, sin; what lies behind the pairs is copied.  The
// gradient is the turn by the negative angle, so one kernel does both.
//
// Bound by memory: every element is read and written once.  The angles are
// formed in fp64 as turns and reduced to half a turn before they are rounded,
// so far positions lose nothing; that costs some forty instructions a pair, so
// a workgroup computes the table of its tokens once, into shared memory, and
// uses it for all heads of q and k.  An item is eight pairs (two 16-byte
// accesses in 16-bit types), or one pair where widths or addresses do not
// allow that.
//
// 4 x 8192 tokens, 32 + 8 heads of 128 bf16: 123 us a direction (5.4 TB/s); 64 x 197 tokens, 12
// heads of 64 fp16: 14.5 us (5.3 TB/s); 32 tokens: 4 us, a launch.

#include <torch/extension.h>
#include <ATen/DeviceGuard.h>
#include <ATen/hip/HIPContext.h>

#include "vec.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 512;   // of a head
constexpr int kMaxTokens = 16;   // of a workgroup
constexpr int kTable = 512;      // pairs of all its tokens, at most

struct Strides { int64_t b, l, h; };

// n / d for n < 2^16 and 0 < d < 2^16 by one multiplication.
struct Divider {
  uint32_t d, m;
  explicit Divider(uint32_t d_) : d(d_), m(d_ == 1 ? 0 : static_cast<uint32_t>(((uint64_t{1} << 32) + d_ - 1) / d_)) {}
  DEVINL uint32_t quotient(uint32_t n) const { return d == 1 ? n : __umulhi(n, m); }
};

struct RotaryArgs {
  const void* q; const void* k; void* qo; void* ko;
  Strides qs, ks;
  const void* pos; bool pos64; int64_t pb, pl, pa;
  const double* freq;
  int n, P, D, Hq, H, tokens_per_block, heads_per_block;  // H: heads of q and k together
  int64_t tokens, L;
  float amplitude, sign;
  Divider per_head, heads;  // items of a head; heads of a token in a block
};

// One rounding fewer than two products and a sum, and the same in every variant.
DEVINL float2 turned(float x, float y, float2 t) {
  return make_float2(fmaf(x, t.x, -(y * t.y)), fmaf(x, t.y, y * t.x));
}

template <typename T, bool VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 table[kTable];
  __shared__ int64_t q_at[kMaxTokens], k_at[kMaxTokens];
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_block;
  const int count = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_block), a.tokens - token0));
  for (int i = threadIdx.x; i < count * a.P; i += kThreads) {
    const int j = i / a.P, pair = i - j * a.P;
    const int64_t b = (token0 + j) / a.L, l = (token0 + j) - b * a.L;
    const int64_t at = b * a.pb + l * a.pl + (pair / a.n) * a.pa;
    const double p = a.pos64 ? static_cast<double>(static_cast<const int64_t*>(a.pos)[at])
                             : static_cast<double>(static_cast<const int32_t*>(a.pos)[at]);
    const double turns = p * a.freq[pair] * 0.15915494309189533577;  // 1 / (2 pi)
    const float half = static_cast<float>(2.0 * (turns - rint(turns)));
    float z, c;
    sincospif(half, &z, &c);
    table[i] = make_float2(c * a.amplitude, z * a.amplitude * a.sign);
    if (pair == 0) {
      q_at[j] = b * a.qs.b + l * a.qs.l;
      k_at[j] = b * a.ks.b + l * a.ks.l;
    }
  }
  __syncthreads();

  constexpr int W = VEC ? 8 : 1;
  const int rot_items = a.P / W;
  const int items = count * a.heads_per_block * a.per_head.d;
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int th = a.per_head.quotient(i);   // token and head
    const int c = i - th * a.per_head.d;
    const int j = a.heads.quotient(th);
    const int h = blockIdx.y * a.heads_per_block + th - j * a.heads_per_block;
    if (h >= a.H) break;  // the last heads' blocks hold one token each
    const bool is_q = h < a.Hq;
    const T* src = is_q ? static_cast<const T*>(a.q) + q_at[j] + h * a.qs.h
                        : static_cast<const T*>(a.k) + k_at[j] + (h - a.Hq) * a.ks.h;
    T* dst = is_q ? static_cast<T*>(a.qo) + ((token0 + j) * a.Hq + h) * a.D
                  : static_cast<T*>(a.ko) + ((token0 + j) * (a.H - a.Hq) + (h - a.Hq)) * a.D;
    if (c >= rot_items) {  // behind the pairs
      const int at = 2 * a.P + (c - rot_items) * W;
      if (VEC) {
        *reinterpret_cast<Vec8<T>*>(dst + at) = *reinterpret_cast<const Vec8<T>*>(src + at);
      } else {
        dst[at] = src[at];
      }
      continue;
    }
    const float2* cz = table + j * a.P + c * W;
    if (VEC) {
      const int at = INTERLEAVED ? c * 16 : c * 8;
      const int other = INTERLEAVED ? at + 8 : at + a.P;
      float x[8], y[8], u[8], v[8];
      load8(src + at, x);
      load8(src + other, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (INTERLEAVED) {
          float& s0 = e < 4 ? x[2 * e] : y[2 * e - 8];
          float& s1 = e < 4 ? x[2 * e + 1] : y[2 * e - 7];
          const float2 r = turned(s0, s1, cz[e]);
          s0 = r.x;
          s1 = r.y;
        } else {
          const float2 r = turned(x[e], y[e], cz[e]);
          u[e] = r.x;
          v[e] = r.y;
        }
      }
      store8(dst + at, INTERLEAVED ? x : u);
      store8(dst + other, INTERLEAVED ? y : v);
    } else {
      const int at = INTERLEAVED ? 2 * c : c;
      const int other = INTERLEAVED ? at + 1 : at + a.P;
      const float2 r = turned(to_f(src[at]), to_f(src[other]), cz[0]);
      dst[at] = from_f<T>(r.x);
      dst[other] = from_f<T>(r.y);
    }
  }
}

void check_heads(const torch::Tensor& x, const torch::Tensor& q) {
  TORCH_CHECK(x.is_cuda() && x.device() == q.device() && x.dim() == 4 && x.size(0) == q.size(0) &&
                  x.size(1) == q.size(1) && x.size(3) == q.size(3) && x.scalar_type() == q.scalar_type() &&
                  (x.stride(3) == 1 || x.size(3) == 1),
              "rotary: q and k are [batch, length, heads, width] of one type on one device, the last stride 1");
}

bool vector_ready(const torch::Tensor& x) {
  const int64_t per16 = 16 / x.element_size();
  return reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && x.stride(0) % per16 == 0 &&
         x.stride(1) % per16 == 0 && x.stride(2) % per16 == 0;
}

}  // namespace

// The turned q (and k), contiguous.  `frequencies`: fp64 [axes * n], radians a
// position; `positions`: int32 or int64 [batch, length, axes].
std::vector<torch::Tensor> rotary_turn(torch::Tensor q, c10::optional<torch::Tensor> k,
                                       torch::Tensor positions, torch::Tensor frequencies,
                                       bool interleaved, double amplitude, bool backward) {
  check_heads(q, q);
  if (k.has_value()) check_heads(*k, q);
  const int64_t B = q.size(0), L = q.size(1), Hq = q.size(2), D = q.size(3);
  const int64_t Hk = k.has_value() ? k->size(2) : 0, P = frequencies.numel();
  TORCH_CHECK(frequencies.device() == q.device() && frequencies.scalar_type() == at::kDouble &&
                  frequencies.is_contiguous() && P >= 1 && P <= kMaxPairs && 2 * P <= D,
              "rotary: 1 to ", kMaxPairs, " frequencies in fp64, two elements of a head each");
  TORCH_CHECK(positions.device() == q.device() && positions.dim() == 3 && positions.size(0) == B &&
                  positions.size(1) == L && positions.size(2) >= 1 && P % positions.size(2) == 0 &&
                  (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong),
              "rotary: positions are int32 or int64 [batch, length, axes]");
  TORCH_CHECK(D <= 4096 && Hq + Hk <= 4096, "rotary: heads too many or too wide");  // and per_head, at most D, under 2^16
  at::DeviceGuard guard(q.device());
  auto qo = torch::empty({B, L, Hq, D}, q.options());
  auto ko = k.has_value() ? torch::empty({B, L, Hk, D}, q.options()) : torch::Tensor();
  std::vector<torch::Tensor> out{qo};
  if (k.has_value()) out.push_back(ko);
  const int64_t tokens = B * L, H = Hq + Hk;
  if (tokens == 0 || H == 0) return out;
  const bool vec = P % 8 == 0 && D % 8 == 0 && vector_ready(q) && (!k.has_value() || vector_ready(*k));
  const int64_t per_head = vec ? P / 8 + (D - 2 * P) / 8 : P + (D - 2 * P);
  // as many tokens as fill the table's 256 threads, fewer where that leaves CUs
  // without work, and items that stay under the divider's 2^16
  const int64_t block_heads = std::min<int64_t>(H, 65535 / per_head);  // a token's heads go over blocks where they are more
  int64_t per_block = std::min<int64_t>({kThreads / std::min<int64_t>(P, kThreads), kMaxTokens,
                                         (tokens + 511) / 512, 65535 / (block_heads * per_head)});
  per_block = block_heads < H ? 1 : std::max<int64_t>(per_block, 1);
  const int64_t blocks = (tokens + per_block - 1) / per_block;
  TORCH_CHECK(launchable(blocks, kThreads), "rotary: too many tokens, ", tokens);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((H + block_heads - 1) / block_heads));
  RotaryArgs a{q.data_ptr(), k.has_value() ? k->data_ptr() : nullptr, qo.data_ptr(),
               k.has_value() ? ko.data_ptr() : nullptr,
               Strides{q.stride(0), q.stride(1), q.stride(2)},
               k.has_value() ? Strides{k->stride(0), k->stride(1), k->stride(2)} : Strides{0, 0, 0},
               positions.data_ptr(), positions.scalar_type() == at::kLong,
               positions.stride(0), positions.stride(1), positions.stride(2),
               frequencies.data_ptr<double>(), static_cast<int>(P / positions.size(2)),
               static_cast<int>(P), static_cast<int>(D), static_cast<int>(Hq), static_cast<int>(H),
               static_cast<int>(per_block), static_cast<int>(block_heads), tokens, L, static_cast<float>(amplitude),
               backward ? -1.f : 1.f, Divider(per_head), Divider(block_heads)};
  auto stream = at::hip::getCurrentHIPStream();
  DISPATCH_FLOAT(q.scalar_type(), "rotary", [&] {
    if (vec) {
      if (interleaved) rotary_kernel<T, true, true><<<grid, kThreads, 0, stream>>>(a);
      else rotary_kernel<T, true, false><<<grid, kThreads, 0, stream>>>(a);
    } else {
      if (interleaved) rotary_kernel<T, false, true><<<grid, kThreads, 0, stream>>>(a);
      else rotary_kernel<T, false, false><<<grid, kThreads, 0, stream>>>(a);
    }
  });
  HIP_CHECK_LAST();
  return out;
}
