// What the attention kernels share: the call, the mask, the score's transform,
// and one row at a time, which every other path falls back to.
//
//   s_ij = scale q_i k_j ; with a cap c: s = c tanh(s / c) ; s -= slope_h |i + off - j|
//   off  = Lk - Lq (the last query stands at the last key)
//   seen = (doc_i == doc_j >= 0) and (not causal or j <= i + off or j < prefix_b)
//   o_i  = sum over seen j of softmax_j(s_ij) v_j, 0 where nothing is seen
//
// Exponents are to the base 2: scores are multiplied by log2(e) once.  The
// statistic kept for the backward pass is lse_i = log2 sum_j 2^(s_ij log2 e),
// +infinity where nothing is seen, so that 2^(s - lse) is 0 there.
#pragma once

#include "vec.h"

constexpr float kLog2e = 1.44269504088896340736f;

struct RowStrides { int64_t b, l, h; };  // elements; the width is contiguous

struct AttnArgs {
  const void* q; const void* k; const void* v;
  RowStrides qs, ks, vs;
  void* o;               // [B, Lq, H, D]
  void* o_rest;          // [B, Lq, H, D] or null: what rounding took from o, for delta
  float* lse;            // [B, H, Lq]
  int B, Lq, Lk, H, Hk, D;
  float scale;
  float softcap;         // 0: none
  const float* slopes;   // [H] or null
  bool causal;
  const int* prefix;     // [B] or null
  const int* q_doc;      // [B, Lq] or null
  const int* k_doc;      // [B, Lk] or null
  const int* q_order;    // [B, blocks of 128 queries] or null: the order to take them in
  const int* k_order;    // the same of keys
  // backward
  const void* dout; RowStrides gs;
  float* delta;          // [B, H, Lq]: sum_d dout o
  // fp16, or null
  float* row_top;        // [B, H, Lq]: the largest finite |dout| of a query
  float* block_top;      // [B, H, blocks of 32 queries]: the largest of those
  float* key_lift;       // [B, Hk, Lk]: what a key's score gradients are multiplied by
  void* dq;              // [B, Lq, H, D]
  void* dk; void* dv;    // [B, Lk, Hk, D]
};

// The first key that a causal query at row i cannot see.
DEVINL int causal_end(const AttnArgs& a, int b, int i) {
  const int end = i + a.Lk - a.Lq + 1;
  return a.prefix != nullptr ? max(end, a.prefix[b]) : end;
}

DEVINL bool seen_by_documents(int dq, int dk) { return dq == dk && dk >= 0; }

// c tanh(x) and the derivative of tanh at x.  16-bit types: with u = 1 / (1 + 2^(2 log2(e) x))
// they are c - 2 c u and 4 u (1 - u), an exponential and a reciprocal, each a unit or so off:
// under 8 units of c together, which with c <= 1024 is half a step of an fp16 weight.  fp32
// takes the library's tanh, whose error is relative to the value.
template <typename T> DEVINL float cap(float x, float c, float& bend) {
  const float u = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.f * kLog2e * x));
  bend = 4.f * fmaf(-u, u, u);
  return fmaf(-2.f * c, u, c);
}
template <> DEVINL float cap<float>(float x, float c, float& bend) {
  const float t = tanhf(x);
  bend = (1.f - t) * (1.f + t);
  return c * t;
}

template <typename T>
DEVINL float dot_row(const T* __restrict__ x, const T* __restrict__ y, int D) {
  float s = 0.f;
  for (int d = 0; d < D; d += 8) {
    float a[8], b[8];
    load8(x + d, a);
    load8(y + d, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(a[e], b[e], s);
  }
  return s;
}

// A score in base 2 and (for the backward pass) the cap's derivative.
template <typename T>
DEVINL float transformed(const AttnArgs& a, float dot, float slope, int distance, float* bend) {
  float s = dot * a.scale;
  *bend = 1.f;
  if (a.softcap > 0.f) s = cap<T>(s / a.softcap, a.softcap, *bend);
  return (s - slope * static_cast<float>(distance)) * kLog2e;
}

// fp16 has 2^-14 for its least normal number, and over long rows weights and score
// gradients lie under it.  Weights are taken times 2^10 in the products over
// queries; score gradients times a power of two that brings the largest |dO| (of the
// query for dQ, of all queries that see the key for dK) to 8 .. 16.  They overflow only
// where weight times sum over the width is 2^12 times the largest |dO|, and then the row
// is done again.  Lower, long rows lose bits: of 32768 even weights dQ was 3.0 times as far
// off as by the result's own rounding with 1/4 .. 1/2, 1.4 times from 4 .. 8 on.
DEVINL float grad_scale(float top) { return top > 0.f ? exp2f(3.f - static_cast<float>(ilogbf(top))) : 1.f; }

// --- one row with one wave: any mask, and nothing that a masked key holds ---

template <typename T>
DEVINL bool row_sees(const AttnArgs& a, int b, int i, int j) {
  if (a.causal && j >= causal_end(a, b, i)) return false;
  if (a.k_doc != nullptr &&
      !seen_by_documents(a.q_doc[static_cast<int64_t>(b) * a.Lq + i], a.k_doc[static_cast<int64_t>(b) * a.Lk + j]))
    return false;
  return true;
}

template <typename T>
DEVINL const T* q_row(const AttnArgs& a, int b, int i, int h) {
  return static_cast<const T*>(a.q) + b * a.qs.b + i * a.qs.l + h * a.qs.h;
}
template <typename T>
DEVINL const T* k_row(const AttnArgs& a, int b, int j, int c) {
  return static_cast<const T*>(a.k) + b * a.ks.b + j * a.ks.l + c * a.ks.h;
}
template <typename T>
DEVINL const T* v_row(const AttnArgs& a, int b, int j, int c) {
  return static_cast<const T*>(a.v) + b * a.vs.b + j * a.vs.l + c * a.vs.h;
}
template <typename T>
DEVINL const T* g_row(const AttnArgs& a, int b, int i, int h) {
  return static_cast<const T*>(a.dout) + b * a.gs.b + i * a.gs.l + h * a.gs.h;
}

DEVINL float lane_of(float v, int lane) { return __shfl(v, lane, WAVE); }

// Whether a row's sums, two of the width a lane, are NaN throughout: they stay so whatever
// follows, and inputs that are NaN everywhere end their rows at once.
DEVINL bool lost(const float (&x)[2], int lane, int D) { return __all((lane >= D || x[0] != x[0]) && (lane + 64 >= D || x[1] != x[1])); }

// Widths up to 128: two elements a lane.
template <typename T>
DEVINL void forward_row(const AttnArgs& a, int b, int i, int h) {
  const int lane = threadIdx.x % WAVE, c = h / (a.H / a.Hk), at = i + a.Lk - a.Lq;
  const float slope = a.slopes != nullptr ? a.slopes[h] : 0.f;
  const T* q = q_row<T>(a, b, i, h);
  float top = -INFINITY, total = 0.f, o[2] = {0.f, 0.f};
  bool none = true;
  for (int j0 = 0; j0 < a.Lk; j0 += WAVE) {
    const int j = j0 + lane;
    const bool sees = j < a.Lk && row_sees<T>(a, b, i, j);
    float s = -INFINITY, bend;
    if (sees) s = transformed<T>(a, dot_row(q, k_row<T>(a, b, j, c), a.D), slope, abs(at - j), &bend);
    uint64_t keys = __ballot(sees);
    if (keys == 0) continue;
    none = false;
    float m = top;
    for (uint64_t left = keys; left != 0; left &= left - 1) {  // NaN stays
      const float x = lane_of(s, __builtin_ctzll(left));
      m = max_or_nan(x, m);
    }
    const float keep = top == -INFINITY ? 0.f : exp2f(top - m);
    const float p = sees ? (m == -INFINITY ? 0.f : exp2f(s - m)) : 0.f;
    top = m;
    total = total * keep + wave_reduce_sum(p);
    o[0] *= keep;
    o[1] *= keep;
    for (; keys != 0; keys &= keys - 1) {
      const int t = __builtin_ctzll(keys);
      const T* v = v_row<T>(a, b, j0 + t, c);
      const float w = lane_of(p, t);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (lane + 64 * x < a.D) o[x] += w * to_f(v[lane + 64 * x]);
    }
    if (total != total && lost(o, lane, a.D)) break;
  }
  const int64_t at_o = ((static_cast<int64_t>(b) * a.Lq + i) * a.H + h) * a.D;
  T* out = static_cast<T*>(a.o) + at_o;
  T* rest = static_cast<T*>(a.o_rest) + at_o;
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (lane + 64 * x < a.D) {
      const float value = none ? 0.f : o[x] / total;
      out[lane + 64 * x] = from_f<T>(value);
      if (a.o_rest != nullptr) rest[lane + 64 * x] = from_f<T>(value - to_f(from_f<T>(value)));
    }
  if (lane == 0) a.lse[(static_cast<int64_t>(b) * a.H + h) * a.Lq + i] = none ? INFINITY : top + log2f(total);
}

template <typename T>
DEVINL void dq_row(const AttnArgs& a, int b, int i, int h, float delta) {
  const int lane = threadIdx.x % WAVE, c = h / (a.H / a.Hk), at = i + a.Lk - a.Lq;
  const float slope = a.slopes != nullptr ? a.slopes[h] : 0.f;
  const float lse = a.lse[(static_cast<int64_t>(b) * a.H + h) * a.Lq + i];
  const T* q = q_row<T>(a, b, i, h);
  const T* g = g_row<T>(a, b, i, h);
  float dq[2] = {0.f, 0.f};
  for (int j0 = 0; j0 < a.Lk; j0 += WAVE) {
    const int j = j0 + lane;
    const bool sees = j < a.Lk && row_sees<T>(a, b, i, j);
    float ds = 0.f;
    if (sees) {
      float bend;
      const float s = transformed<T>(a, dot_row(q, k_row<T>(a, b, j, c), a.D), slope, abs(at - j), &bend);
      ds = exp2f(s - lse) * (dot_row(g, v_row<T>(a, b, j, c), a.D) - delta) * bend * a.scale;
    }
    for (uint64_t keys = __ballot(sees); keys != 0; keys &= keys - 1) {
      const int t = __builtin_ctzll(keys);
      const T* k = k_row<T>(a, b, j0 + t, c);
      const float w = lane_of(ds, t);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (lane + 64 * x < a.D) dq[x] += w * to_f(k[lane + 64 * x]);
    }
    if (lost(dq, lane, a.D)) break;
  }
  T* out = static_cast<T*>(a.dq) + ((static_cast<int64_t>(b) * a.Lq + i) * a.H + h) * a.D;
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (lane + 64 * x < a.D) out[lane + 64 * x] = from_f<T>(dq[x]);
}

template <typename T>
DEVINL void dkv_row(const AttnArgs& a, int b, int j, int c) {
  const int lane = threadIdx.x % WAVE, group = a.H / a.Hk;
  const T* k = k_row<T>(a, b, j, c);
  const T* v = v_row<T>(a, b, j, c);
  float dk[2] = {0.f, 0.f}, dv[2] = {0.f, 0.f};
  bool all = false;
  for (int h = c * group; h < (c + 1) * group && !all; ++h) {
    const float slope = a.slopes != nullptr ? a.slopes[h] : 0.f;
    for (int i0 = 0; i0 < a.Lq && !all; i0 += WAVE) {
      const int i = i0 + lane;
      const bool sees = i < a.Lq && row_sees<T>(a, b, i, j);
      float p = 0.f, ds = 0.f;
      if (sees) {
        const int64_t stat = (static_cast<int64_t>(b) * a.H + h) * a.Lq + i;
        float bend;
        const float s = transformed<T>(a, dot_row(q_row<T>(a, b, i, h), k, a.D), slope, abs(i + a.Lk - a.Lq - j), &bend);
        p = exp2f(s - a.lse[stat]);
        ds = p * (dot_row(g_row<T>(a, b, i, h), v, a.D) - a.delta[stat]) * bend * a.scale;
      }
      for (uint64_t rows = __ballot(sees); rows != 0; rows &= rows - 1) {
        const int t = __builtin_ctzll(rows);
        const T* q = q_row<T>(a, b, i0 + t, h);
        const T* g = g_row<T>(a, b, i0 + t, h);
        const float wp = lane_of(p, t), ws = lane_of(ds, t);
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (lane + 64 * x < a.D) {
            dk[x] += ws * to_f(q[lane + 64 * x]);
            dv[x] += wp * to_f(g[lane + 64 * x]);
          }
      }
      all = lost(dk, lane, a.D) && lost(dv, lane, a.D);
    }
  }
  const int64_t out = ((static_cast<int64_t>(b) * a.Lk + j) * a.Hk + c) * a.D;
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (lane + 64 * x < a.D) {
      static_cast<T*>(a.dk)[out + lane + 64 * x] = from_f<T>(dk[x]);
      static_cast<T*>(a.dv)[out + lane + 64 * x] = from_f<T>(dv[x]);
    }
}
