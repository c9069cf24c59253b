// Element types and eight-element vectors of the transformer kernels (gfx950).
//
// Every kernel here computes in fp32 and touches memory in groups of eight
// elements: 16 bytes of bf16 / fp16, 32 bytes of fp32 (two 16-byte accesses).
#pragma once

#include "common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

using bf16_t = __bf16;
using fp16_t = _Float16;

template <typename T> DEVINL float to_f(T v) { return static_cast<float>(v); }

// Round to nearest, ties to even, in every type.
template <typename T> DEVINL T from_f(float v) { return static_cast<T>(v); }

template <typename T>
struct alignas(16) Vec8 {
  T v[8];
};

template <typename T>
DEVINL void load8(const T* __restrict__ p, float (&out)[8]) {
  const Vec8<T> x = *reinterpret_cast<const Vec8<T>*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = to_f(x.v[i]);
}

template <typename T>
DEVINL void store8(T* __restrict__ p, const float (&in)[8]) {
  Vec8<T> x;
#pragma unroll
  for (int i = 0; i < 8; ++i) x.v[i] = from_f<T>(in[i]);
  *reinterpret_cast<Vec8<T>*>(p) = x;
}

// Four fp32 values as four e4m3 codes (round to nearest even; NaN stays NaN).
// The caller has brought them into [-448, 448].
DEVINL uint32_t pack_fp8(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

// The larger of two magnitudes; NaN if one of them is.
DEVINL float max_or_nan(float a, float b) { return (a > b || a != a) ? a : b; }

// Whether a launch fits: beyond 2^32 - 1 threads along x the runtime starts the rest of the
// division, and says nothing.
inline bool launchable(int64_t blocks, int64_t threads) { return blocks * threads < (int64_t{1} << 32); }

// Runs `fn` with a value of the element type that `dtype` names.
#define DISPATCH_FLOAT(dtype, NAME, ...)                                   \
  [&] {                                                                    \
    switch (dtype) {                                                       \
      case at::kFloat: { using T = float; return __VA_ARGS__(); }          \
      case at::kBFloat16: { using T = bf16_t; return __VA_ARGS__(); }      \
      case at::kHalf: { using T = fp16_t; return __VA_ARGS__(); }          \
      default: TORCH_CHECK(false, NAME ": fp32, bf16 or fp16 expected, got ", dtype); \
    }                                                                      \
  }()
