// Attention with capped scores, distance biases and masks: forward and backward
// (gfx950).  The mathematics stands in attention.h.

#include <torch/extension.h>
#include <ATen/DeviceGuard.h>
#include <ATen/hip/HIPContext.h>

#include "attention_tile.h"

namespace {
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / WAVE;
constexpr int kQueries = 32 * kWaves;  // of a workgroup of the tiled kernels
constexpr float kLazy = 8.f;           // how far a maximum may rise before sums are scaled down

// --- ids of 64 rows ---------------------------------------------------------

__global__ __launch_bounds__(WAVE) void doc_ranges_kernel(const int* __restrict__ ids, int L, int tiles,
                                                          DocRange* __restrict__ out) {
  const int b = blockIdx.x / tiles, t = blockIdx.x % tiles, row = t * kDocTile + threadIdx.x;
  const int id = row < L ? ids[static_cast<int64_t>(b) * L + row] : -1;
  const int lo = wave_min(id >= 0 ? id : INT_MAX), hi = wave_max(id);
  const bool one = __ballot(id >= 0 && lo == hi) == ~uint64_t{0};
  if (threadIdx.x == 0) out[blockIdx.x] = DocRange{lo, hi, one, 0};
}

// The keys before which the query of a lane sees any (0: none), and its id.
struct Query {
  int at, end, doc;
  float slope2;  // times log2(e)
};

DEVINL Query query_of(const AttnArgs& a, int b, int i, int h, bool ok) {
  Query q;
  q.at = i + a.Lk - a.Lq;
  q.doc = ok && a.q_doc != nullptr ? a.q_doc[static_cast<int64_t>(b) * a.Lq + i] : 0;
  q.end = !ok || q.doc < 0 ? 0 : a.causal ? max(0, min(a.Lk, causal_end(a, b, i))) : a.Lk;
  q.slope2 = ok && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
  return q;
}

// Scores in registers to base-2 scores: on return a score is s * (the returned
// factor).  Lanes are queries and registers keys: `first` is the key of register 0
// of half 0.  `bend`: the cap's derivative, for the backward pass.
template <typename T, bool BEND>
DEVINL float transform(const AttnArgs& a, f32x16& s, f32x16* bend, int first, int at, float slope2, bool as_is) {
  const float c = fabsf(a.scale) * kLog2e;
  if (as_is) return c;
  const int half = threadIdx.x % WAVE / 32;
  if (a.softcap > 0.f) {
    const float in = fabsf(a.scale) / a.softcap, out = a.softcap * kLog2e;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float t = tanh_of<T>(s[r] * in);
      s[r] = out * t;
      if (BEND) (*bend)[r] = 1.f - t * t;
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= c;
  }
  if (a.slopes != nullptr) {
    const float d0 = static_cast<float>(at - first - 4 * half);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] -= slope2 * fabsf(d0 - static_cast<float>(result_row(r, 0)));
  }
  return 1.f;
}

// Whether scores go to the exponent with one factor.
DEVINL bool plain_scores(const AttnArgs& a) { return !(a.softcap > 0.f) && a.slopes == nullptr && a.scale != 0.f; }

// Which registers a query sees, as bits.
DEVINL uint32_t seen_keys(const AttnArgs& a, const Query& q, const int* kd, int first, int row0) {
  const int half = threadIdx.x % WAVE / 32, left = q.end - first - 4 * half;
  uint32_t seen = 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) seen |= static_cast<uint32_t>(result_row(r, 0) < left) << r;
  if (a.k_doc != nullptr) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int4 d = *reinterpret_cast<const int4*>(kd + row0 + 8 * x + 4 * half);
      const uint32_t same = static_cast<uint32_t>(d.x == q.doc) | static_cast<uint32_t>(d.y == q.doc) << 1 |
                            static_cast<uint32_t>(d.z == q.doc) << 2 | static_cast<uint32_t>(d.w == q.doc) << 3;
      seen &= same << (4 * x) | ~(15u << (4 * x));
    }
  }
  return seen;
}

// --- forward ----------------------------------------------------------------

// The running softmax of 32 queries (a lane and its other half hold one) and
// their outputs, transposed: columns are queries, rows the width.  `l` is the
// lane's own part of the sum.  `top` may lag behind the true maximum by kLazy, so
// that weights reach 2^kLazy and the outputs are scaled only where it rises more.
template <typename T, int DP, int NS>
struct Online {
  using Tl = Tile<T, DP>;
  f32x16 o[DP / 32];
  float top, l;

  DEVINL void clear() {
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) o[x] = zeros16();
    top = -INFINITY;
    l = 0.f;
  }

  DEVINL void absorb(const AttnArgs& a, const Frag<T> (&qf)[DP / 16], const T* ks, const T* vs, const int* kd,
                     const Query& q, int first, bool masked) {
    f32x16 s[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      s[n] = zeros16();
#pragma unroll
      for (int step = 0; step < DP / 16; ++step) product(Tl::rows(ks, 32 * n, step), qf[step], s[n]);
    }
    const bool as_is = plain_scores(a);
    float c = 1.f, high = -INFINITY;
#pragma unroll
    for (int n = 0; n < NS; ++n) c = transform<T, false>(a, s[n], nullptr, first + 32 * n, q.at, q.slope2, as_is);
    if (masked) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const uint32_t seen = seen_keys(a, q, kd, first + 32 * n, 32 * n);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = (seen >> r & 1) ? s[n][r] : -INFINITY;
      }
    }
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) high = fmaxf(high, s[n][r]);
    high = fmaxf(high, other_half(high)) * c;
    if (__any(high > top + kLazy)) {
      const float now = fmaxf(top, high);
      const float keep = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
      top = now;
      l *= keep;
#pragma unroll
      for (int x = 0; x < DP / 32; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[x][r] *= keep;
    }
    const float from = top == -INFINITY ? 0.f : top;
    Frag<T> p[NS][2];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[n][r], c, -from));
        l += w;
        p[n][r / 8].set(r % 8, w);
      }
#pragma unroll
    for (int x = 0; x < DP / 32; ++x)
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t) product(Tl::columns(vs, 32 * n + 16 * t, 32 * x), p[n][t], o[x]);
  }
};

// Four neighbouring elements of a row.
template <typename T>
DEVINL void store4(T* p, float a, float b, float c, float d) {
  struct alignas(4 * sizeof(T)) Four { T v[4]; };
  *reinterpret_cast<Four*>(p) = Four{{from_f<T>(a), from_f<T>(b), from_f<T>(c), from_f<T>(d)}};
}

// A lane's column of a transposed result times `by`, to the row at `out`.
template <typename T, int DP>
DEVINL void store_column(T* out, const f32x16 (&o)[DP / 32], int D, float by) {
  const int half = threadIdx.x % WAVE / 32;
#pragma unroll
  for (int x = 0; x < DP / 32; ++x)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * x + result_row(r, half);
      if (d < D) store4(out + d, o[x][r] * by, o[x][r + 1] * by, o[x][r + 2] * by, o[x][r + 3] * by);
    }
}

template <int N>
DEVINL bool finite_column(const f32x16 (&o)[N]) {
  bool fine = true;
#pragma unroll
  for (int x = 0; x < N; ++x)
#pragma unroll
    for (int r = 0; r < 16; ++r) fine = fine && fabsf(o[x][r]) <= FLT_MAX;
  return fine;
}

// Of 32 columns, which have a value that is not finite in either half.
DEVINL uint32_t bad_columns(bool bad) {
  const uint64_t both = __ballot(bad);
  return static_cast<uint32_t>(both) | static_cast<uint32_t>(both >> 32);
}

// Rows that come out not finite are done again one by one: a matrix product
// multiplies what a masked place holds by zero, and NaN or infinity there spoils
// the sum; an fp16 operand may overflow.  Without masks and in types of fp32's
// range the value is the formula's own.
template <typename T>
DEVINL bool repairs(const AttnArgs& a) { return sizeof(T) == 2 || a.causal || a.k_doc != nullptr; }

template <typename T, int DP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void forward_tiles_kernel(AttnArgs a, const DocRange* ranges, int q_tiles) {
  constexpr int KT = sizeof(T) == 2 ? 64 : 32, NS = KT / 32;
  __shared__ __attribute__((aligned(16))) T ks[2][KT * DP];
  __shared__ __attribute__((aligned(16))) T vs[2][KT * DP];
  __shared__ __attribute__((aligned(16))) int kd[2][KT];
  const int t = threadIdx.x, lane = t % WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(t / WAVE);
  const int64_t linear = xcd_order(blockIdx.x, gridDim.x);
  const int64_t bh = linear / q_tiles;
  const int i0 = (q_tiles - 1 - static_cast<int>(linear % q_tiles)) * kQueries;
  const int b = bh / a.H, h = bh % a.H, kv = h / (a.H / a.Hk);
  const int i = i0 + 32 * wave + lane % 32;
  const bool ok = i < a.Lq;
  const Query q = query_of(a, b, i, h, ok);
  Frag<T> qf[DP / 16];
  load_operands<T, DP>(q_row<T>(a, b, ok ? i : 0, h), ok, a.D, qf);
  if (a.scale < 0.f) {
#pragma unroll
    for (int x = 0; x < DP / 16; ++x) qf[x].v = -qf[x].v;
  }
  const int least_end = wave_min(q.end), most_end = wave_max(q.end);
  const int doc_lo = wave_min(q.doc), doc_hi = wave_max(q.doc);

  int lo = 0, hi = 0;  // ids of the workgroup's queries
  if (ranges != nullptr) {
    lo = INT_MAX, hi = -1;
#pragma unroll
    for (int x = 0; x < kQueries; x += WAVE)
      if (i0 + x + lane < a.Lq) {
        const int id = a.q_doc[static_cast<int64_t>(b) * a.Lq + i0 + x + lane];
        if (id >= 0) lo = min(lo, id);
        hi = max(hi, id);
      }
    lo = wave_min(lo), hi = wave_max(hi);
  }
  const int j_end = a.causal ? max(0, min(a.Lk, causal_end(a, b, min(i0 + kQueries, a.Lq) - 1))) : a.Lk;
  const int k_tiles = (a.Lk + kDocTile - 1) / kDocTile;
  const DocRange* own = ranges != nullptr ? ranges + static_cast<int64_t>(b) * k_tiles : nullptr;
  TileWalk walk(own, lo, hi, 0, (j_end + kDocTile - 1) / kDocTile);
  int rest = -1;  // the second half of a tile of ids where a tile of keys is smaller
  auto next = [&]() {
    if (KT < kDocTile && rest >= 0) {
      const int j = rest;
      rest = -1;
      return j;
    }
    const int n = walk.next();
    if (n < 0) return -1;
    if (KT < kDocTile && n * kDocTile + KT < j_end) rest = n * kDocTile + KT;
    return n * kDocTile;
  };
  const T* k0 = k_row<T>(a, b, 0, kv);
  const T* v0 = v_row<T>(a, b, 0, kv);
  const int* d0 = a.k_doc != nullptr ? a.k_doc + static_cast<int64_t>(b) * a.Lk : nullptr;

  Online<T, DP, NS> run;
  run.clear();
  Staged<T, DP, KT, kThreads> sk, sv;
  int sd = -1;
  auto load = [&](int j) {
    sk.load(k0 + j * a.ks.l, a.ks.l, a.Lk - j, a.D, d0 != nullptr ? d0 + j : nullptr, t);
    sv.load(v0 + j * a.vs.l, a.vs.l, a.Lk - j, a.D, d0 != nullptr ? d0 + j : nullptr, t);
    if (d0 != nullptr && t < KT) sd = j + t < a.Lk ? d0[j + t] : -1;
  };
  auto store = [&](int buf) {
    sk.store(ks[buf], t);
    sv.store(vs[buf], t);
    if (d0 != nullptr && t < KT) kd[buf][t] = sd;
  };
  int j = next(), buf = 0;
  if (j >= 0) {
    load(j);
    store(0);
  }
  __syncthreads();
  while (j >= 0) {
    const int following = next();
    if (following >= 0) load(following);
    if (j < most_end) {
      bool masked = j + KT > least_end;
      if (own != nullptr) {
        const DocRange r = own[j / kDocTile];
        masked = masked || !(r.one && doc_lo == doc_hi && r.lo == doc_lo);
      }
      run.absorb(a, qf, ks[buf], vs[buf], kd[buf], q, j, masked);
    }
    if (following >= 0) store(buf ^ 1);
    __syncthreads();
    j = following;
    buf ^= 1;
  }

  const float total = run.l + other_half(run.l);
  const bool none = run.top == -INFINITY && !(total != total);
  uint32_t again = 0;
  if (repairs<T>(a)) again = bad_columns(ok && (!finite_column(run.o) || !(fabsf(total) <= FLT_MAX)));
  if (ok && !(again >> (lane % 32) & 1)) {
    const float by = none ? 0.f : 1.f / total;
    store_column<T, DP>(static_cast<T*>(a.o) + ((static_cast<int64_t>(b) * a.Lq + i) * a.H + h) * a.D, run.o, a.D, by);
    if (lane < 32) a.lse[bh * a.Lq + i] = none ? INFINITY : run.top + log2f(total);
  }
  for (; again != 0; again &= again - 1) forward_row<T>(a, b, i0 + 32 * wave + __builtin_ctz(again), h);
}

// --- backward ---------------------------------------------------------------

// dQ of 32 queries a wave: lanes are queries, K and V pass by in tiles.
//   P^T = 2^(S^T - lse), dS^T = P^T (V dO^T - delta) bend, dQ^T += K^T dS^T
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void dq_tiles_kernel(AttnArgs a, const DocRange* ranges, int q_tiles) {
  constexpr int KT = sizeof(T) == 2 ? 64 : 32;
  using Tl = Tile<T, DP>;
  __shared__ __attribute__((aligned(16))) T ks[2][KT * DP];
  __shared__ __attribute__((aligned(16))) T vs[2][KT * DP];
  __shared__ __attribute__((aligned(16))) int kd[2][KT];
  const int t = threadIdx.x, lane = t % WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(t / WAVE);
  const int64_t linear = xcd_order(blockIdx.x, gridDim.x);
  const int64_t bh = linear / q_tiles;
  const int i0 = (q_tiles - 1 - static_cast<int>(linear % q_tiles)) * kQueries;
  const int b = bh / a.H, h = bh % a.H, kv = h / (a.H / a.Hk);
  const int i = i0 + 32 * wave + lane % 32;
  const bool ok = i < a.Lq;
  const Query q = query_of(a, b, i, h, ok);
  Frag<T> qf[DP / 16], gf[DP / 16];
  load_operands<T, DP>(q_row<T>(a, b, ok ? i : 0, h), ok, a.D, qf);
  load_operands<T, DP>(g_row<T>(a, b, ok ? i : 0, h), ok, a.D, gf);
  if (a.scale < 0.f) {
#pragma unroll
    for (int x = 0; x < DP / 16; ++x) qf[x].v = -qf[x].v;
  }
  const float lse = ok ? a.lse[bh * a.Lq + i] : INFINITY, delta = ok ? a.delta[bh * a.Lq + i] : 0.f;
  const int least_end = wave_min(q.end), most_end = wave_max(q.end);
  const int doc_lo = wave_min(q.doc), doc_hi = wave_max(q.doc);
  int lo = 0, hi = 0;
  if (ranges != nullptr) {
    lo = INT_MAX, hi = -1;
#pragma unroll
    for (int x = 0; x < kQueries; x += WAVE)
      if (i0 + x + lane < a.Lq) {
        const int id = a.q_doc[static_cast<int64_t>(b) * a.Lq + i0 + x + lane];
        if (id >= 0) lo = min(lo, id);
        hi = max(hi, id);
      }
    lo = wave_min(lo), hi = wave_max(hi);
  }
  const int j_end = a.causal ? max(0, min(a.Lk, causal_end(a, b, min(i0 + kQueries, a.Lq) - 1))) : a.Lk;
  const int k_tiles = (a.Lk + kDocTile - 1) / kDocTile;
  const DocRange* own = ranges != nullptr ? ranges + static_cast<int64_t>(b) * k_tiles : nullptr;
  TileWalk walk(own, lo, hi, 0, (j_end + kDocTile - 1) / kDocTile);
  int rest = -1;
  auto next = [&]() {
    if (KT < kDocTile && rest >= 0) {
      const int j = rest;
      rest = -1;
      return j;
    }
    const int n = walk.next();
    if (n < 0) return -1;
    if (KT < kDocTile && n * kDocTile + KT < j_end) rest = n * kDocTile + KT;
    return n * kDocTile;
  };
  const T* k0 = k_row<T>(a, b, 0, kv);
  const T* v0 = v_row<T>(a, b, 0, kv);
  const int* d0 = a.k_doc != nullptr ? a.k_doc + static_cast<int64_t>(b) * a.Lk : nullptr;
  const bool as_is = plain_scores(a);

  f32x16 dq[DP / 32];
#pragma unroll
  for (int x = 0; x < DP / 32; ++x) dq[x] = zeros16();
  Staged<T, DP, KT, kThreads> sk, sv;
  int sd = -1;
  auto load = [&](int j) {
    sk.load(k0 + j * a.ks.l, a.ks.l, a.Lk - j, a.D, d0 != nullptr ? d0 + j : nullptr, t);
    sv.load(v0 + j * a.vs.l, a.vs.l, a.Lk - j, a.D, d0 != nullptr ? d0 + j : nullptr, t);
    if (d0 != nullptr && t < KT) sd = j + t < a.Lk ? d0[j + t] : -1;
  };
  auto store = [&](int buf) {
    sk.store(ks[buf], t);
    sv.store(vs[buf], t);
    if (d0 != nullptr && t < KT) kd[buf][t] = sd;
  };
  int j = next(), buf = 0;
  if (j >= 0) {
    load(j);
    store(0);
  }
  __syncthreads();
  while (j >= 0) {
    const int following = next();
    if (following >= 0) load(following);
    if (j < most_end) {
      bool masked = j + KT > least_end;
      if (own != nullptr) {
        const DocRange r = own[j / kDocTile];
        masked = masked || !(r.one && doc_lo == doc_hi && r.lo == doc_lo);
      }
#pragma unroll
      for (int n = 0; n < KT / 32; ++n) {
        f32x16 s = zeros16(), dp = zeros16(), bend;
#pragma unroll
        for (int step = 0; step < DP / 16; ++step) {
          product(Tl::rows(ks[buf], 32 * n, step), qf[step], s);
          product(Tl::rows(vs[buf], 32 * n, step), gf[step], dp);
        }
        const float c = transform<T, true>(a, s, &bend, j + 32 * n, q.at, q.slope2, as_is);
        uint32_t seen = 0xFFFF;
        if (masked) seen = seen_keys(a, q, kd[buf], j + 32 * n, 32 * n);
        Frag<T> ds[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float x = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * (dp[r] - delta);
          if (a.softcap > 0.f) x *= bend[r];
          ds[r / 8].set(r % 8, (seen >> r & 1) ? x : 0.f);
        }
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
#pragma unroll
          for (int u = 0; u < 2; ++u) product(Tl::columns(ks[buf], 32 * n + 16 * u, 32 * x), ds[u], dq[x]);
      }
    }
    if (following >= 0) store(buf ^ 1);
    __syncthreads();
    j = following;
    buf ^= 1;
  }
  uint32_t again = 0;
  if (repairs<T>(a)) again = bad_columns(ok && !finite_column(dq));
  if (ok && !(again >> (lane % 32) & 1))
    store_column<T, DP>(static_cast<T*>(a.dq) + ((static_cast<int64_t>(b) * a.Lq + i) * a.H + h) * a.D, dq, a.D, a.scale);
  for (; again != 0; again &= again - 1) dq_row<T>(a, b, i0 + 32 * wave + __builtin_ctz(again), h);
}

// dK and dV of 32 keys a wave: lanes are keys, Q and dO of all heads that share
// them pass by in tiles.
//   P = 2^(S - lse), dV^T += dO^T P, dS = P (dO V^T - delta) bend, dK^T += Q^T dS
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 && DP == 64 ? 2 : 1) void dkv_tiles_kernel(AttnArgs a, const DocRange* ranges, int k_blocks) {
  constexpr int QT = sizeof(T) == 2 ? 64 : 32, kKeys = 32 * kWaves;
  using Tl = Tile<T, DP>;
  __shared__ __attribute__((aligned(16))) T qs[2][QT * DP];
  __shared__ __attribute__((aligned(16))) T gs[2][QT * DP];
  __shared__ __attribute__((aligned(16))) float stats[2][2][QT];  // lse, delta
  __shared__ __attribute__((aligned(16))) int qd[2][QT];
  const int t = threadIdx.x, lane = t % WAVE, half = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(t / WAVE);
  const int64_t linear = xcd_order(blockIdx.x, gridDim.x);
  const int64_t bc = linear / k_blocks;
  const int j0 = static_cast<int>(linear % k_blocks) * kKeys;
  const int b = bc / a.Hk, kv = bc % a.Hk, group = a.H / a.Hk, off = a.Lk - a.Lq;
  const int j = j0 + 32 * wave + lane % 32;
  const int doc = j < a.Lk && a.k_doc != nullptr ? a.k_doc[static_cast<int64_t>(b) * a.Lk + j] : 0;
  const bool in = j < a.Lk, ok = in && doc >= 0;
  Frag<T> kf[DP / 16], vf[DP / 16];
  load_operands<T, DP>(k_row<T>(a, b, ok ? j : 0, kv), ok, a.D, kf);
  load_operands<T, DP>(v_row<T>(a, b, ok ? j : 0, kv), ok, a.D, vf);
  if (a.scale < 0.f) {
#pragma unroll
    for (int x = 0; x < DP / 16; ++x) kf[x].v = -kf[x].v;
  }
  // the first query that sees a key
  const int prefix = a.prefix != nullptr ? a.prefix[b] : 0;
  const int begin = !ok ? INT_MAX : !a.causal || j < prefix ? 0 : max(0, j - off);
  const int least_begin = wave_min(begin), most_begin = wave_max(begin);
  const int doc_lo = wave_min(doc), doc_hi = wave_max(doc);
  int lo = 0, hi = 0;
  if (ranges != nullptr) {
    lo = INT_MAX, hi = -1;
#pragma unroll
    for (int x = 0; x < kKeys; x += WAVE)
      if (j0 + x + lane < a.Lk) {
        const int id = a.k_doc[static_cast<int64_t>(b) * a.Lk + j0 + x + lane];
        if (id >= 0) lo = min(lo, id);
        hi = max(hi, id);
      }
    lo = wave_min(lo), hi = wave_max(hi);
  }
  const int i_begin = !a.causal || j0 < prefix ? 0 : max(0, j0 - off);
  const int q_tiles = (a.Lq + kDocTile - 1) / kDocTile;
  const DocRange* own = ranges != nullptr ? ranges + static_cast<int64_t>(b) * q_tiles : nullptr;
  int head = kv * group, rest = -1;
  TileWalk walk(own, lo, hi, i_begin / kDocTile, q_tiles);
  auto next = [&](int& at_head) {
    if (QT < kDocTile && rest >= 0) {
      const int i = rest;
      rest = -1;
      at_head = head;
      return i;
    }
    int n = walk.next();
    while (n < 0) {
      if (++head == (kv + 1) * group) return -1;
      walk = TileWalk(own, lo, hi, i_begin / kDocTile, q_tiles);
      n = walk.next();
      if (n < 0) return -1;  // none for one head: none for any
    }
    if (QT < kDocTile && n * kDocTile + QT < a.Lq) rest = n * kDocTile + QT;
    at_head = head;
    return n * kDocTile;
  };
  const bool as_is = plain_scores(a);
  const int* d0 = a.q_doc != nullptr ? a.q_doc + static_cast<int64_t>(b) * a.Lq : nullptr;

  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int x = 0; x < DP / 32; ++x) dk[x] = zeros16(), dv[x] = zeros16();
  Staged<T, DP, QT, kThreads> sq, sg;
  float stat = 0.f;
  int sd = -1;
  auto load = [&](int i, int h) {
    sq.load(q_row<T>(a, b, i, h), a.qs.l, a.Lq - i, a.D, d0 != nullptr ? d0 + i : nullptr, t);
    sg.load(g_row<T>(a, b, i, h), a.gs.l, a.Lq - i, a.D, d0 != nullptr ? d0 + i : nullptr, t);
    const int64_t at = (static_cast<int64_t>(b) * a.H + h) * a.Lq + i;
    if (t < QT) stat = i + t < a.Lq ? a.lse[at + t] : INFINITY;
    else if (t < 2 * QT) stat = i + t - QT < a.Lq ? a.delta[at + t - QT] : 0.f;
    if (d0 != nullptr && t < QT) sd = i + t < a.Lq ? d0[i + t] : -1;
  };
  auto store = [&](int buf) {
    sq.store(qs[buf], t);
    sg.store(gs[buf], t);
    if (t < 2 * QT) stats[buf][t / QT][t % QT] = stat;
    if (d0 != nullptr && t < QT) qd[buf][t] = sd;
  };
  int h = head, h_next = head, buf = 0;
  int i = next(h);
  if (i >= 0) {
    load(i, h);
    store(0);
  }
  __syncthreads();
  while (i >= 0) {
    const int following = next(h_next);
    if (following >= 0) load(following, h_next);
    if (i + QT > least_begin) {
      const float slope2 = a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
      bool masked = i < most_begin;
      if (own != nullptr) {
        const DocRange r = own[i / kDocTile];
        masked = masked || !(r.one && doc_lo == doc_hi && r.lo == doc_lo);
      }
#pragma unroll
      for (int n = 0; n < QT / 32; ++n) {
        f32x16 s = zeros16(), dp = zeros16(), bend;
#pragma unroll
        for (int step = 0; step < DP / 16; ++step) {
          product(Tl::rows(qs[buf], 32 * n, step), kf[step], s);
          product(Tl::rows(gs[buf], 32 * n, step), vf[step], dp);
        }
        // the distance |i + off - j| with queries in registers: as if the key stood at j - off
        const float c = transform<T, true>(a, s, &bend, i + 32 * n, j - off, slope2, as_is);
        uint32_t seen = 0xFFFF;
        if (masked) {
          seen = 0;
          const int from = begin == INT_MAX ? INT_MAX : begin - i - 32 * n - 4 * half;
#pragma unroll
          for (int r = 0; r < 16; ++r) seen |= static_cast<uint32_t>(result_row(r, 0) >= from) << r;
          if (d0 != nullptr) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int4 d = *reinterpret_cast<const int4*>(&qd[buf][32 * n + 8 * x + 4 * half]);
              const uint32_t same = static_cast<uint32_t>(d.x == doc) | static_cast<uint32_t>(d.y == doc) << 1 |
                                    static_cast<uint32_t>(d.z == doc) << 2 | static_cast<uint32_t>(d.w == doc) << 3;
              seen &= same << (4 * x) | ~(15u << (4 * x));
            }
          }
        }
        Frag<T> p[2], ds[2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 lse = *reinterpret_cast<const float4*>(&stats[buf][0][32 * n + 8 * x + 4 * half]);
          const float4 del = *reinterpret_cast<const float4*>(&stats[buf][1][32 * n + 8 * x + 4 * half]);
          const float ls[4] = {lse.x, lse.y, lse.z, lse.w}, de[4] = {del.x, del.y, del.z, del.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int r = 4 * x + y;
            const float w = __builtin_amdgcn_exp2f(fmaf(s[r], c, -ls[y]));
            float g = w * (dp[r] - de[y]);
            if (a.softcap > 0.f) g *= bend[r];
            const bool sees = seen >> r & 1;
            p[r / 8].set(r % 8, sees ? w : 0.f);
            ds[r / 8].set(r % 8, sees ? g : 0.f);
          }
        }
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            product(Tl::columns(gs[buf], 32 * n + 16 * u, 32 * x), p[u], dv[x]);
            product(Tl::columns(qs[buf], 32 * n + 16 * u, 32 * x), ds[u], dk[x]);
          }
      }
    }
    if (following >= 0) store(buf ^ 1);
    __syncthreads();
    i = following;
    h = h_next;
    buf ^= 1;
  }
  uint32_t again = 0;
  if (repairs<T>(a)) again = bad_columns(in && !(finite_column(dk) && finite_column(dv)));
  if (in && !(again >> (lane % 32) & 1)) {
    const int64_t out = ((static_cast<int64_t>(b) * a.Lk + j) * a.Hk + kv) * a.D;
    store_column<T, DP>(static_cast<T*>(a.dk) + out, dk, a.D, a.scale);
    store_column<T, DP>(static_cast<T*>(a.dv) + out, dv, a.D, 1.f);
  }
  for (; again != 0; again &= again - 1) dkv_row<T>(a, b, j0 + 32 * wave + __builtin_ctz(again), kv);
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
  TORCH_CHECK(x.size(1) <= 1 || x.stride(1) * x.element_size() <= (1 << 24), "attention: rows of ", name, " lie over 16 MB apart");
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

// The ids of every 64 rows, or nothing.
torch::Tensor doc_ranges(const c10::optional<torch::Tensor>& ids, int B, int L, hipStream_t stream) {
  if (!ids.has_value()) return torch::Tensor();
  const int tiles = (L + kDocTile - 1) / kDocTile;
  auto out = torch::empty({static_cast<int64_t>(B) * tiles, 4}, ids->options());
  doc_ranges_kernel<<<blocks_for(static_cast<int64_t>(B) * tiles, 1), WAVE, 0, stream>>>(
      ids->data_ptr<int>(), L, tiles, reinterpret_cast<DocRange*>(out.data_ptr<int>()));
  HIP_CHECK_LAST();
  return out;
}

const DocRange* ranges_of(const torch::Tensor& x) {
  return x.defined() ? reinterpret_cast<const DocRange*>(x.data_ptr<int>()) : nullptr;
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
  const auto ranges = doc_ranges(k_doc, a.B, a.Lk, stream);
  const int q_tiles = (a.Lq + kQueries - 1) / kQueries;
  const int grid = blocks_for(static_cast<int64_t>(a.B) * a.H * q_tiles, 1);
  DISPATCH_FLOAT(q.scalar_type(), "attention", [&] {
    if (a.D <= 64) forward_tiles_kernel<T, 64><<<grid, kThreads, 0, stream>>>(a, ranges_of(ranges), q_tiles);
    else forward_tiles_kernel<T, 128><<<grid, kThreads, 0, stream>>>(a, ranges_of(ranges), q_tiles);
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
  const auto k_ranges = doc_ranges(k_doc, a.B, a.Lk, stream), q_ranges = doc_ranges(q_doc, a.B, a.Lq, stream);
  const int64_t rows = static_cast<int64_t>(a.B) * a.H * a.Lq;
  const int q_tiles = (a.Lq + kQueries - 1) / kQueries, k_blocks = (a.Lk + kQueries - 1) / kQueries;
  const int q_grid = blocks_for(static_cast<int64_t>(a.B) * a.H * q_tiles, 1);
  const int k_grid = blocks_for(static_cast<int64_t>(a.B) * a.Hk * k_blocks, 1);
  DISPATCH_FLOAT(q.scalar_type(), "attention", [&] {
    delta_kernel<T><<<blocks_for(rows, kThreads / 16), kThreads, 0, stream>>>(a, delta.data_ptr<float>(), rows);
    if (a.D <= 64) {
      dq_tiles_kernel<T, 64><<<q_grid, kThreads, 0, stream>>>(a, ranges_of(k_ranges), q_tiles);
      dkv_tiles_kernel<T, 64><<<k_grid, kThreads, 0, stream>>>(a, ranges_of(q_ranges), k_blocks);
    } else {
      dq_tiles_kernel<T, 128><<<q_grid, kThreads, 0, stream>>>(a, ranges_of(k_ranges), q_tiles);
      dkv_tiles_kernel<T, 128><<<k_grid, kThreads, 0, stream>>>(a, ranges_of(q_ranges), k_blocks);
    }
  });
  HIP_CHECK_LAST();
  return {dq, dk, dv};
}
