// The attention kernels and how they are launched, for one element type a source
// file (gfx950).  The mathematics stands in attention.h.
#pragma once

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include "attention_tile.h"
#include "attention_launch.h"

namespace {
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / WAVE;
constexpr int kQueries = 32 * kWaves;  // of a workgroup of the tiled kernels
static_assert(kQueries == 2 * kDocTile, "blocks of rows are ordered by pairs of tiles");

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

// What scores go through, as a constant of the kernel, so that products and
// exponentials are one block of instructions: nothing (one factor, not zero), the
// cap, a bias (or a factor of zero), both.
enum Score { kPlain, kCapped, kBiased, kBoth };
constexpr bool capped(Score s) { return s == kCapped || s == kBoth; }

// A score in a register to one in base 2 (a kPlain one still wants the factor).
// Lanes are queries and registers keys, or the other way round: only the distance
// matters.
template <typename T, Score SC>
struct ScoreMap {
  float factor;  // of the exponent's argument
  float in, out, slope2, d0;

  // `apart`: what the lane's index is ahead of the first register's of half 0.
  DEVINL ScoreMap(const AttnArgs& a, float slope, int apart) {
    // not 0: what is not seen is -infinity here, and 0 times that is not a number
    const float c = fmaxf(fabsf(a.scale) * kLog2e, FLT_MIN);
    factor = SC == kPlain ? c : 1.f;
    in = capped(SC) ? fabsf(a.scale) / a.softcap : c;
    out = a.softcap * kLog2e;
    slope2 = slope;
    d0 = static_cast<float>(apart - 4 * (static_cast<int>(threadIdx.x) % WAVE / 32));
  }

  // Register r; `bend` gets the cap's derivative.
  DEVINL float operator()(float s, int r, float& bend) const {
    bend = 1.f;
    if (SC == kPlain) return s;
    if (capped(SC)) {
      s = cap<T>(s * in, out, bend);
    } else {
      s *= in;
    }
    if (SC == kBiased || SC == kBoth) s -= slope2 * fabsf(d0 - static_cast<float>(result_row(r, 0)));
    return s;
  }
};

// What a tile's masks ask of every pair: no question, an end (or a beginning), an id as
// well.
enum Mask { kSeen, kEnds, kIds };

// Which of the pairs (lane, register) are seen.  `left`: registers' rows before it,
// from half 0 on; with FROM, rows from it on.  `ids`: of the registers' rows; `doc`: the
// lane's, one that no row has if it is negative.
template <Mask MASK, bool FROM>
struct Seen {
  int bound, doc;
  const int* ids;
  int4 four;

  DEVINL Seen(int bound_, int doc_, const int* ids_) {
    const int half = threadIdx.x % WAVE / 32;
    bound = bound_ - 4 * half;
    doc = doc_ < 0 ? -2 : doc_;
    ids = ids_ + 4 * half;
  }

  DEVINL bool operator()(int r) {
    bool ok = FROM ? result_row(r, 0) >= bound : result_row(r, 0) < bound;
    if (MASK == kIds) {
      if (r % 4 == 0) four = *reinterpret_cast<const int4*>(ids + 2 * r);
      ok = ok && (r % 4 == 0 ? four.x : r % 4 == 1 ? four.y : r % 4 == 2 ? four.z : four.w) == doc;
    }
    return ok;
  }
};

// x, or 0 where bit r is not set.
DEVINL float with_bit(float x, uint32_t bits, int r) {
  return __uint_as_float(__float_as_uint(x) & static_cast<uint32_t>(static_cast<int32_t>(bits << (31 - r)) >> 31));
}

// --- forward ----------------------------------------------------------------

// The running softmax of 32 queries (a lane and its other half hold one) and
// their outputs, transposed: columns are queries, rows the width.  `l` is the
// lane's own part of the sum.  The outputs are scaled at every tile: a branch around
// that made the compiler keep them twice.
template <typename T, int DP, int NS>
struct Online {
  f32x16 o[DP / 32];
  float top, l;
  bool by_id;  // with documents: whether this half has seen a key

  DEVINL void clear() {
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) o[x] = zeros16();
    top = -INFINITY;
    l = 0.f;
    by_id = false;
  }

  // Whether the query sees any key: its scores may all be -infinity, which is no reason for zeros.
  DEVINL bool sees(const AttnArgs& a, const Query& q) const {
    const bool other = __shfl_xor(static_cast<int>(by_id), 32, WAVE) != 0;
    return a.k_doc == nullptr ? q.end > 0 : by_id || other;
  }

  template <Score SC>
  DEVINL void absorb(const AttnArgs& a, const Reader<T, DP>& reader, const Frag<T> (&qf)[DP / 16], const T* ks, const T* vs, const int* kd,
                     const Query& q, int first, Mask mask) {
    const Reader<T, DP> at = reader.fresh();
    Frag<T> p[NS][2];
    f32x16 s[NS];
    scores(at, qf, ks, s);
    weights<SC>(a, s, p, kd, q, first, mask);
    outputs(at, vs, p);
  }

  static DEVINL void scores(const Reader<T, DP>& at, const Frag<T> (&qf)[DP / 16], const T* ks, f32x16 (&s)[NS]) {
    constexpr int kSteps = DP / 16;
#pragma unroll
    for (int n = 0; n < NS; ++n) s[n] = zeros16();
    piped<T, NS * kSteps, 4>([&](auto i) { return at.rows(ks, 32 * (i / kSteps), i % kSteps); },
                             [&](auto i, const Frag<T>& k) { product(k, qf[i % kSteps], s[i / kSteps]); });
  }

  template <Score SC>
  DEVINL void weights(const AttnArgs& a, f32x16 (&s)[NS], Frag<T> (&p)[NS][2], const int* kd, const Query& q, int first, Mask mask) {
    float c = 1.f, high = -INFINITY;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const ScoreMap<T, SC> map(a, q.slope2, q.at - first - 32 * n);
      c = map.factor;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float bend;
        s[n][r] = map(s[n][r], r, bend);
      }
    }
    auto apply = [&](auto which) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        Seen<decltype(which)::value, false> seen(q.end - first - 32 * n, q.doc, kd + 32 * n);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool ok = seen(r);
          s[n][r] = ok ? s[n][r] : -INFINITY;
          if (decltype(which)::value == kIds) by_id = by_id || ok;
        }
      }
    };
    if (mask == kSeen) by_id = true;
    if (mask == kEnds) apply(std::integral_constant<Mask, kEnds>());
    if (mask == kIds) apply(std::integral_constant<Mask, kIds>());
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) high = fmaxf(high, s[n][r]);
    high = fmaxf(high, other_half(high)) * c;
    const float now = fmaxf(top, high), from = now == -INFINITY ? 0.f : now;
    const float keep = __builtin_amdgcn_exp2f(top - from);
    top = now;
    l *= keep;
#pragma unroll
    for (int x = 0; x < DP / 32; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[x][r] *= keep;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float w0 = __builtin_amdgcn_exp2f(fmaf(s[n][r], c, -from)), w1 = __builtin_amdgcn_exp2f(fmaf(s[n][r + 1], c, -from));
        l += w0 + w1;
        p[n][r / 8].set2(r % 8, w0, w1);
      }
  }

  DEVINL void outputs(const Reader<T, DP>& at, const T* vs, const Frag<T> (&p)[NS][2]) {
    constexpr int kWide = DP / 32;
    piped<T, NS * 2 * kWide, 4>([&](auto i) { return at.columns(vs, 16 * (i / kWide), i % kWide); },
                                [&](auto i, const Frag<T>& v) { product(v, p[i / kWide / 2][i / kWide % 2], o[i % kWide]); });
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

// What rounding takes from them.
template <typename T, int DP>
DEVINL void store_rest(T* out, const f32x16 (&o)[DP / 32], int D, float by) {
  const int half = threadIdx.x % WAVE / 32;
#pragma unroll
  for (int x = 0; x < DP / 32; ++x)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * x + result_row(r, half);
      float e[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float value = o[x][r + y] * by;
        e[y] = value - to_f(from_f<T>(value));
      }
      if (d < D) store4(out + d, e[0], e[1], e[2], e[3]);
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
DEVINL bool repairs(const AttnArgs& a) { return std::is_same<T, fp16_t>::value || a.causal || a.k_doc != nullptr; }

// 32 queries a wave: S^T = K Q^T with lanes as queries, so that a row's maximum and sum stay
// in a lane and its half, and P^T is the operand of O^T = V^T P^T as it lies.  128 queries a
// workgroup read each key tile once; two tiles in shared memory, one in use, and three
// workgroups of width 64 a CU (two of 128).  Bound by the vector units at width 64 (an
// exponential and seven more instructions a score; 48% of the time, products 15%), which a
// wave's waits leave idle, and by the products at width 128.  64 images of 197 tokens, 12
// heads of 64 bf16: 36 us; 8191 tokens, 16 heads of 128 fp16, causal: 371 us, 744 TFLOP/s.
template <typename T, int DP, Score SC>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? (DP == 64 ? 3 : 2) : 1) void forward_tiles_kernel(AttnArgs a, const DocRange* ranges, int q_tiles) {
  constexpr int KT = sizeof(T) == 2 ? 64 : 32, NS = KT / 32;
  __shared__ __attribute__((aligned(16))) T ks[2][KT * DP];
  __shared__ __attribute__((aligned(16))) T vs[2][KT * DP];
  __shared__ __attribute__((aligned(16))) int kd[2][KT];
  const int t = threadIdx.x, lane = t % WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(t / WAVE);
  const int64_t linear = xcd_order(blockIdx.x, gridDim.x);
  int64_t bh = linear / q_tiles;
  int i0 = tile_at(linear % q_tiles, q_tiles, bh, a.causal && a.k_doc == nullptr) * kQueries;
  if (a.q_order != nullptr) i0 = ordered(a.q_order, linear, q_tiles, a.B, a.H, bh) * kQueries;
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
  // rows that are not there decide nothing, and nothing of them is kept
  const int least_end = wave_min(ok ? q.end : INT_MAX), most_end = wave_max(q.end);
  const int doc_lo = wave_min(ok ? q.doc : INT_MAX), doc_hi = wave_max(ok ? q.doc : INT_MIN);
  const int doc_least = doc_lo >= 0 ? doc_lo : wave_min(ok && q.doc >= 0 ? q.doc : INT_MAX);

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

  const Reader<T, DP> at;
  Online<T, DP, NS> run;
  run.clear();
  uint32_t ids = 0;
  DocRange range{0, 0, 0}, range_next{0, 0, 0};
  uint64_t there = 0;
  auto load = [&](int j, auto buf) {
    there = first_rows(a.Lk - j);
    if (own != nullptr) {
      range_next = walk.of(j / kDocTile);
      there = range_next.there >> (j % kDocTile);
      ids = staged_word(d0 + j, t, min(KT, a.Lk - j));
    }
    Flight<T, DP, KT, kWaves>::load(k0 + j * a.ks.l, a.ks.l, there, a.D, ks[buf], wave);
    Flight<T, DP, KT, kWaves>::load(v0 + j * a.vs.l, a.vs.l, there, a.D, vs[buf], wave);
  };
  auto landed = [&](auto buf) {  // what load() began is there for all waves
    if (own != nullptr && t < KT) kd[buf][t] = (there >> t & 1) ? static_cast<int>(ids) : -1;
    range = range_next;
    arrived<0>();
    __syncthreads();
  };
  // One tile is used while the next is on its way into the other buffer.
  int j = next();
  auto turn = [&](auto buf) {
    constexpr int kBuf = decltype(buf)::value;
    const int following = next();
    const DocRange present = range;
    if (following >= 0) load(following, std::integral_constant<int, 1 - kBuf>());
    if (j < most_end && (own == nullptr || (present.lo <= doc_hi && present.hi >= doc_least))) {
      bool masked = j + KT > least_end;
      if (own != nullptr) masked = masked || !(present.one() && doc_lo == doc_hi && present.lo == doc_lo);
      run.template absorb<SC>(a, at, qf, ks[kBuf], vs[kBuf], kd[kBuf], q, j, !masked ? kSeen : own == nullptr ? kEnds : kIds);
    }
    landed(std::integral_constant<int, 1 - kBuf>());
    j = following;
  };
  if (j >= 0) {
    load(j, std::integral_constant<int, 0>());
    landed(std::integral_constant<int, 0>());
    do {
      turn(std::integral_constant<int, 0>());
      if (j >= 0) turn(std::integral_constant<int, 1>());
    } while (j >= 0);
  }

  const float total = run.l + other_half(run.l);
  const bool none = !run.sees(a, q);
  uint32_t again = 0;
  if (repairs<T>(a)) again = bad_columns(ok && (!finite_column(run.o) || !(fabsf(total) <= FLT_MAX)));
  if (ok && !(again >> (lane % 32) & 1)) {
    const float by = none ? 0.f : 1.f / total;
    const int64_t to = ((static_cast<int64_t>(b) * a.Lq + i) * a.H + h) * a.D;
    store_column<T, DP>(static_cast<T*>(a.o) + to, run.o, a.D, by);
    if (a.o_rest != nullptr) store_rest<T, DP>(static_cast<T*>(a.o_rest) + to, run.o, a.D, by);
    if (lane < 32) a.lse[bh * a.Lq + i] = none ? INFINITY : run.top + log2f(total);
  }
  for (; again != 0; again &= again - 1) forward_row<T>(a, b, i0 + 32 * wave + __builtin_ctz(again), h);
}

// In place of the sum of weights, which is not negative, of a part in which a row sees no key.
constexpr float kSeesNone = -1.f;

// One row's joined sums (two of the width a lane), by one wave: the quotient, or
// the row again where it is not finite.
template <typename T>
DEVINL void finish_row(const AttnArgs& a, int b, int i, int h, float o0, float o1, float top, float total, bool none) {
  const int lane = threadIdx.x % WAVE;
  if (repairs<T>(a) && __any(!(fabsf(o0) <= FLT_MAX && fabsf(o1) <= FLT_MAX && fabsf(total) <= FLT_MAX))) {
    forward_row<T>(a, b, i, h);
    return;
  }
  const float by = none ? 0.f : 1.f / total;
  T* out = static_cast<T*>(a.o) + ((static_cast<int64_t>(b) * a.Lq + i) * a.H + h) * a.D;
  o0 *= by, o1 *= by;
  if (lane < a.D) out[lane] = from_f<T>(o0);
  if (lane + 64 < a.D) out[lane + 64] = from_f<T>(o1);
  if (a.o_rest != nullptr) {
    T* rest = static_cast<T*>(a.o_rest) + ((static_cast<int64_t>(b) * a.Lq + i) * a.H + h) * a.D;
    if (lane < a.D) rest[lane] = from_f<T>(o0 - to_f(from_f<T>(o0)));
    if (lane + 64 < a.D) rest[lane + 64] = from_f<T>(o1 - to_f(from_f<T>(o1)));
  }
  if (lane == 0) a.lse[(static_cast<int64_t>(b) * a.H + h) * a.Lq + i] = none ? INFINITY : top + log2f(total);
}

// Few queries: a workgroup takes 32 rows (queries of all heads that share a key
// head) and a stretch of keys, its waves every fourth 32 keys of it, each with
// shared memory of its own, so that nothing waits but for its own loads: as soon as the
// scores have read K's tile the next is on its way to its place.  The waves join at the
// end; where keys are split over workgroups too, `part` [splits, rows, DP] and `stats`
// (maximum, sum) go to the joining kernel.  Bound by memory: 16 caches of up to 65536 keys, 8
// key heads of 128 bf16, are read at 4.9 TB/s (405 us, as fast as a large copy).
template <typename T, int DP, Score SC>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void forward_split_kernel(
    AttnArgs a, const DocRange* ranges, int row_tiles, int splits, int keys_per_split, float* __restrict__ part, float2* __restrict__ stats) {
  constexpr int KT = 32, kPad = DP + 1;
  constexpr int kTileBytes = 2 * kWaves * KT * DP * sizeof(T), kJoinBytes = kWaves * 32 * kPad * 4;
  __shared__ __attribute__((aligned(16))) char shared[kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes];
  __shared__ __attribute__((aligned(16))) int kd[kWaves][KT];
  __shared__ float tops[kWaves][32], totals[kWaves][32];
  const int lane = threadIdx.x % WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  T* ks = reinterpret_cast<T*>(shared) + wave * 2 * KT * DP;
  T* vs = ks + KT * DP;

  int64_t linear = blockIdx.x;  // key heads, whose rows are neighbours in memory, change fastest
  const int kv = linear % a.Hk;
  linear /= a.Hk;
  const int row0 = static_cast<int>(linear % row_tiles) * 32;
  linear /= row_tiles;
  const int split = linear % splits, b = linear / splits;
  const int group = a.H / a.Hk, rows = group * a.Lq;
  const int row = row0 + lane % 32;
  const bool ok = row < rows;
  const int h = kv * group + (ok ? row / a.Lq : 0), i = ok ? row % a.Lq : 0;
  const Query q = query_of(a, b, i, h, ok);
  Frag<T> qf[DP / 16];
  load_operands<T, DP>(q_row<T>(a, b, i, h), ok, a.D, qf);
  if (a.scale < 0.f) {
#pragma unroll
    for (int x = 0; x < DP / 16; ++x) qf[x].v = -qf[x].v;
  }
  const int least_end = wave_min(ok ? q.end : INT_MAX), most_end = wave_max(q.end);
  const int doc_lo = wave_min(ok ? q.doc : INT_MAX), doc_hi = wave_max(ok ? q.doc : INT_MIN);
  const int k_tiles = (a.Lk + kDocTile - 1) / kDocTile;
  const DocRange* own = ranges != nullptr ? ranges + static_cast<int64_t>(b) * k_tiles : nullptr;
  const int* d0 = a.k_doc != nullptr ? a.k_doc + static_cast<int64_t>(b) * a.Lk : nullptr;
  const T* k0 = k_row<T>(a, b, 0, kv);
  const T* v0 = v_row<T>(a, b, 0, kv);
  const int stop = min(most_end, (split + 1) * keys_per_split);

  const Reader<T, DP> at;
  Online<T, DP, 1> run;
  run.clear();
  uint32_t ids = 0;
  DocRange range{0, 0, 0}, range_next{0, 0, 0};
  uint64_t there = 0;
  // This wave's next 32 keys: tiles of 64 that may hold ids of its rows go round by
  // halves, two waves a tile.
  TileWalk walk(own, doc_lo, doc_hi, split * keys_per_split / kDocTile, (stop + kDocTile - 1) / kDocTile);
  int skip = wave / 2;
  auto seek = [&]() {
    for (; skip > 0; --skip)
      if (walk.next() < 0) return stop;
    skip = kWaves / 2 - 1;
    const int n = walk.next();
    if (n < 0) return stop;
    if (own != nullptr) range_next = walk.of(n);
    return min(n * kDocTile + wave % 2 * KT, stop);
  };
  using Way = Flight<T, DP, KT, 1>;
  auto load_k = [&](int j) {
    there = first_rows(a.Lk - j);
    if (own != nullptr) {
      there = range_next.there >> (j % kDocTile);
      ids = staged_word(d0 + j, lane, min(KT, a.Lk - j));
    }
    Way::load(k0 + j * a.ks.l, a.ks.l, there, a.D, ks, 0);
  };
  auto load_v = [&](int j) { Way::load(v0 + j * a.vs.l, a.vs.l, there, a.D, vs, 0); };
  // K of the next tile is asked for as soon as the scores have read this one's, V as
  // soon as the outputs have, so that half to all of a tile is always on its way.
  int j = seek();
  if (j < stop) {
    load_k(j);
    load_v(j);
  }
  while (j < stop) {
    if (own != nullptr && lane < KT) kd[wave][lane] = (there >> lane & 1) ? static_cast<int>(ids) : -1;
    range = range_next;
    const int following = seek();
    Frag<T> p[1][2];
    f32x16 s[1];
    arrived<Way::kLoads>();  // K; V may still come
    run.scores(at, qf, ks, s);
    read_out();
    if (following < stop) load_k(following);
    bool masked = j + KT > least_end;
    if (own != nullptr) masked = masked || !(range.one() && doc_lo == doc_hi && range.lo == doc_lo);
    run.template weights<SC>(a, s, p, kd[wave], q, j, !masked ? kSeen : own == nullptr ? kEnds : kIds);
    if (following < stop) arrived<Way::kLoads>();
    else arrived<0>();
    run.outputs(at, vs, p);
    read_out();
    if (following < stop) load_v(following);
    j = following;
  }

  const float sum_here = run.l + other_half(run.l);
  const float total = run.sees(a, q) ? sum_here : kSeesNone;
  if (lane < 32) tops[wave][lane] = run.top, totals[wave][lane] = total;
  __syncthreads();  // all tiles are used: their memory takes the sums
  float* join = reinterpret_cast<float*>(shared);
#pragma unroll
  for (int x = 0; x < DP / 32; ++x)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      join[(wave * 32 + lane % 32) * kPad + 32 * x + result_row(r, lane / 32)] = run.o[x][r];
  __syncthreads();
  for (int c = wave; c < 32 && row0 + c < rows; c += kWaves) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w][c]);
    float sum = 0.f, o0 = 0.f, o1 = 0.f;
    bool none = true;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float keep = tops[w][c] == -INFINITY && top != -INFINITY ? 0.f : tops[w][c] == top ? 1.f : __builtin_amdgcn_exp2f(tops[w][c] - top);
      if (totals[w][c] != kSeesNone) none = false, sum += keep * totals[w][c];
      o0 += keep * join[(w * 32 + c) * kPad + lane % DP];
      if (DP > 64) o1 += keep * join[(w * 32 + c) * kPad + 64 + lane];
    }
    const int which = row0 + c;
    if (splits == 1) {
      finish_row<T>(a, b, which % a.Lq, kv * group + which / a.Lq, o0, o1, top, sum, none);
    } else {
      const int64_t to = ((static_cast<int64_t>(split) * a.B + b) * a.Hk + kv) * rows + which;
      part[to * DP + lane] = o0;
      if (DP > 64) part[to * DP + 64 + lane] = o1;
      if (lane == 0) stats[to] = make_float2(top, none ? kSeesNone : sum);
    }
  }
}

// Joins the splits of a row: a wave a row, at most 64 splits.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void join_splits_kernel(AttnArgs a, int splits, int64_t count, const float* __restrict__ part,
                                                               const float2* __restrict__ stats) {
  const int lane = threadIdx.x % WAVE;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / WAVE;
  if (at >= count) return;
  const float2 own = lane < splits ? stats[lane * count + at] : make_float2(-INFINITY, kSeesNone);
  float top = own.x;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, WAVE));
  const float keep = own.x == -INFINITY && top != -INFINITY ? 0.f : own.x == top ? 1.f : __builtin_amdgcn_exp2f(own.x - top);
  const bool none = __all(own.y == kSeesNone);
  const float sum = wave_reduce_sum(own.y == kSeesNone ? 0.f : keep * own.y);
  float o0 = 0.f, o1 = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float k = lane_of(keep, s);
    o0 += k * part[(s * count + at) * DP + lane];
    if (DP > 64) o1 += k * part[(s * count + at) * DP + 64 + lane];
  }
  const int rows = a.H / a.Hk * a.Lq, row = at % rows;
  const int64_t bc = at / rows;
  finish_row<T>(a, bc / a.Hk, row % a.Lq, bc % a.Hk * (a.H / a.Hk) + row / a.Lq, o0, o1, top, sum, none);
}

// --- backward ---------------------------------------------------------------

// dQ of 32 queries a wave, and delta for both: lanes are queries, K and V pass by in
// tiles.
//   P^T = 2^(S^T - lse), dS^T = P^T (V dO^T - delta) bend, dQ^T += K^T dS^T
// A kernel of its own and not sums of dK's workgroups into dQ: those would have to be atomic,
// in an order that changes, or another pass.  It costs two of seven products.  64 images of
// 197 tokens, 12 heads of 64 bf16: 46 us; 8191 tokens, 16 heads of 128 fp16, causal: 427 us,
// 969 TFLOP/s, of 1091 in a large library product.
template <typename T, int DP, Score SC, bool FINE>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void dq_tiles_kernel(AttnArgs a, const DocRange* ranges, int q_tiles) {
  constexpr int KT = sizeof(T) == 2 && DP == 64 ? 64 : 32;
  __shared__ __attribute__((aligned(16))) T ks[2][KT * DP];
  __shared__ __attribute__((aligned(16))) T vs[2][KT * DP];
  __shared__ __attribute__((aligned(16))) int kd[2][KT];
  const int t = threadIdx.x, lane = t % WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(t / WAVE);
  const int64_t linear = xcd_order(blockIdx.x, gridDim.x);
  int64_t bh = linear / q_tiles;
  int i0 = tile_at(linear % q_tiles, q_tiles, bh, a.causal && a.k_doc == nullptr) * kQueries;
  if (a.q_order != nullptr) i0 = ordered(a.q_order, linear, q_tiles, a.B, a.H, bh) * kQueries;
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
  // delta = sum_d dO o, with what o's rounding left: it is subtracted from every dP of a
  // row, so that its error does not average out.  With o in 16 bits dQ and dK of short rows
  // are further off: 2.27 times as far as by their own rounding with 2 keys a row, where they
  // are 1.53 with the rest, 1.80 : 1.49 with 4, 1.56 : 1.47 with 16, 1.44 : 1.42 with 197, in
  // bf16 and fp16 alike.  Rows of packed documents are that short in long calls too.
  float delta = 0.f, high = 0.f;
  {
    const int64_t row = ((static_cast<int64_t>(b) * a.Lq + (ok ? i : 0)) * a.H + h) * a.D;
    Frag<T> of[DP / 16], rest[DP / 16];
    load_operands<T, DP>(static_cast<const T*>(a.o) + row, ok, a.D, of);
    load_operands<T, DP>(static_cast<const T*>(a.o_rest) + row, ok && a.o_rest != nullptr, a.D, rest);
#pragma unroll
    for (int x = 0; x < DP / 16; ++x)
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const float g = to_f(gf[x].v[y]);
        delta = fmaf(g, to_f(of[x].v[y]) + to_f(rest[x].v[y]), delta);
        if (std::is_same<T, fp16_t>::value && fabsf(g) <= FLT_MAX) high = fmaxf(high, fabsf(g));
      }
    delta += other_half(delta);
    if (ok && lane < 32) a.delta[bh * a.Lq + i] = delta;
  }
  // dS of fp16 is scaled into its range (see grad_scale), through the exponent
  float lift = 1.f;
  if constexpr (std::is_same<T, fp16_t>::value) {
    high = fmaxf(high, other_half(high));
    lift = grad_scale(high);
    if (ok && lane < 32) a.row_top[bh * a.Lq + i] = high;
    high = wave_reduce_max(high);
    if (lane == 0 && ok) a.block_top[bh * ((a.Lq + 31) / 32) + i / 32] = high;
  }
  const float lse = ok ? a.lse[bh * a.Lq + i] - log2f(lift) : INFINITY;
  // rows that are not there decide nothing, and nothing of them is kept
  const int least_end = wave_min(ok ? q.end : INT_MAX), most_end = wave_max(q.end);
  const int doc_lo = wave_min(ok ? q.doc : INT_MAX), doc_hi = wave_max(ok ? q.doc : INT_MIN);
  const int doc_least = doc_lo >= 0 ? doc_lo : wave_min(ok && q.doc >= 0 ? q.doc : INT_MAX);
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

  f32x16 dq[DP / 32];
#pragma unroll
  for (int x = 0; x < DP / 32; ++x) dq[x] = zeros16();
  const Reader<T, DP> reader;
  // With registers for two sets, the scores of 32 keys pass under the weights of the 32
  // before, and those' products under the weights of these; with one, the other wave
  // of the SIMD has to fill the time.
  constexpr int kSub = KT / 32, kSteps = DP / 16, kWide = DP / 32;
  auto step = [&](bool masked, int j, auto buf) {
    const Reader<T, DP> at = reader.fresh();
    f32x16 s[kSub], dp[kSub];
    Frag<T> ds[kSub][2], rest[FINE ? kSub : 1][2];
    auto score = [&](int n, int i, const Frag<T>& f) {
      if (i == 0) s[n] = zeros16(), dp[n] = zeros16();
      if (i % 2 == 0) product(f, qf[i / 2], s[n]);
      else product(f, gf[i / 2], dp[n]);
    };
    auto score_read = [&](int n, int i) { return at.rows(i % 2 == 0 ? ks[buf] : vs[buf], 32 * n, i / 2); };
    auto output = [&](int n, int i, const Frag<T>& f) {
      product(f, ds[n][i / kWide], dq[i % kWide]);
      if constexpr (FINE) product(f, rest[n][i / kWide], dq[i % kWide]);
    };
    auto output_read = [&](int n, int i) { return at.columns(ks[buf], 32 * n + 16 * (i / kWide), i % kWide); };
    uint32_t bits[kSub];  // one body for all tiles, as for dK and dV
    auto mask = [&](int n) {
      bits[n] = ~0u;
      auto apply = [&](auto which) {
        Seen<decltype(which)::value, false> seen(q.end - j - 32 * n, q.doc, kd[buf] + 32 * n);
        if (capped(SC)) bits[n] = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (capped(SC)) bits[n] |= static_cast<uint32_t>(seen(r)) << r;
          else s[n][r] = seen(r) ? s[n][r] : -INFINITY;
        }
      };
      if (masked && own == nullptr) apply(std::integral_constant<Mask, kEnds>());
      if (masked && own != nullptr) apply(std::integral_constant<Mask, kIds>());
    };
    auto weight = [&](int n, int r) {  // registers r and r + 1, in their order
      const ScoreMap<T, SC> map(a, q.slope2, q.at - j - 32 * n);
      float x[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float bend;
        const float t = map(s[n][r + y], r + y, bend);
        x[y] = __builtin_amdgcn_exp2f(fmaf(t, map.factor, -lse));
        if (capped(SC)) x[y] = with_bit(x[y], bits[n], r + y);
        x[y] *= dp[n][r + y] - delta;
        if (capped(SC)) x[y] *= bend;
      }
      ds[n][r / 8].set2(r % 8, x[0], x[1]);
      if constexpr (FINE) rest[n][r / 8].set2(r % 8, x[0] - to_f(ds[n][r / 8].v[r % 8]), x[1] - to_f(ds[n][r / 8].v[r % 8 + 1]));
    };
    constexpr int kA = 2 * kSteps, kB = 2 * kWide;  // products of scores and of outputs
    if constexpr (kSub == 2 && DP == 64) {
      piped<T, kA, 4>([&](auto i) { return score_read(0, i); }, [&](auto i, const Frag<T>& f) { score(0, i, f); });
      mask(0);
      piped<T, kA, 4>([&](auto i) { return score_read(1, i); },
                      [&](auto i, const Frag<T>& f) {
                        score(1, i, f);
#pragma unroll
                        for (int r = 16 / kA * i; r < 16 / kA * (i + 1); r += 2) weight(0, r);
                      });
      mask(1);
      piped<T, 2 * kB, 4>([&](auto i) { return output_read(i / kB, i % kB); },
                          [&](auto i, const Frag<T>& f) {
                            output(i / kB, i % kB, f);
                            if (i < kB)
#pragma unroll
                              for (int r = 16 / kB * i; r < 16 / kB * (i + 1); r += 2) weight(1, r);
                          });
    } else {
      each(std::make_integer_sequence<int, kSub>(), [&](auto n) {
        piped<T, kA, 4>([&](auto i) { return score_read(n, i); }, [&](auto i, const Frag<T>& f) { score(n, i, f); });
        mask(n);
#pragma unroll
        for (int r = 0; r < 16; r += 2) weight(n, r);
        __builtin_amdgcn_sched_barrier(0);
        piped<T, kB, 4>([&](auto i) { return output_read(n, i); }, [&](auto i, const Frag<T>& f) { output(n, i, f); });
      });
    }
  };
  uint32_t ids = 0;
  DocRange range{0, 0, 0}, range_next{0, 0, 0};
  uint64_t there = 0;
  auto load = [&](int j, auto buf) {
    there = first_rows(a.Lk - j);
    if (own != nullptr) {
      range_next = walk.of(j / kDocTile);
      there = range_next.there >> (j % kDocTile);
      ids = staged_word(d0 + j, t, min(KT, a.Lk - j));
    }
    Flight<T, DP, KT, kWaves>::load(k0 + j * a.ks.l, a.ks.l, there, a.D, ks[buf], wave);
    Flight<T, DP, KT, kWaves>::load(v0 + j * a.vs.l, a.vs.l, there, a.D, vs[buf], wave);
  };
  auto landed = [&](auto buf) {  // what load() began is there for all waves
    if (own != nullptr && t < KT) kd[buf][t] = (there >> t & 1) ? static_cast<int>(ids) : -1;
    range = range_next;
    arrived<0>();
    __syncthreads();
  };
  // One tile is used while the next is on its way into the other buffer.
  int j = next();
  auto turn = [&](auto buf) {
    constexpr int kBuf = decltype(buf)::value;
    const int following = next();
    const DocRange present = range;
    if (following >= 0) load(following, std::integral_constant<int, 1 - kBuf>());
    if (j < most_end && (own == nullptr || (present.lo <= doc_hi && present.hi >= doc_least))) {
      bool masked = j + KT > least_end;
      if (own != nullptr) masked = masked || !(present.one() && doc_lo == doc_hi && present.lo == doc_lo);
      step(masked, j, buf);
    }
    landed(std::integral_constant<int, 1 - kBuf>());
    j = following;
  };
  if (j >= 0) {
    load(j, std::integral_constant<int, 0>());
    landed(std::integral_constant<int, 0>());
    do {
      turn(std::integral_constant<int, 0>());
      if (j >= 0) turn(std::integral_constant<int, 1>());
    } while (j >= 0);
  }

  uint32_t again = 0;
  if (repairs<T>(a)) again = bad_columns(ok && !finite_column(dq));
  if (ok && !(again >> (lane % 32) & 1))
    store_column<T, DP>(static_cast<T*>(a.dq) + ((static_cast<int64_t>(b) * a.Lq + i) * a.H + h) * a.D, dq, a.D, a.scale / lift);
  for (; again != 0; again &= again - 1)
    dq_row<T>(a, b, i0 + 32 * wave + __builtin_ctz(again), h, lane_of(delta, __builtin_ctz(again)));
}

// dK and dV of 32 keys a wave: lanes are keys, Q and dO of all heads that share
// them pass by in tiles.
//   P = 2^(S - lse), dV^T += dO^T P, dS = P (dO V^T - delta) bend, dK^T += Q^T dS
// Bound by registers: both sums, and K's and V's operands, are 192 of a wave's 256 at width
// 128, and what is left sets how far reads and weights go ahead of the products.  64 images of
// 197 tokens, 12 heads of 64 bf16: 51 us; 8191 tokens, 16 heads on 4 of 128 fp16, causal:
// 706 us, 782 TFLOP/s, of 1091 in a large library product, and 55 us for the join of eight
// parts (4.5 TB/s).
template <typename T, int DP, Score SC, bool FINE>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void dkv_tiles_kernel(AttnArgs a, const DocRange* ranges, int k_blocks, int splits, float* __restrict__ part) {
  constexpr bool kHalf = sizeof(T) == 2 && DP == 128;
  constexpr int QT = sizeof(T) == 2 && DP == 64 ? 64 : 32, kKeys = 32 * kWaves;
  // Width 128 in 16 bits fits two waves a SIMD with V's operands and some of K's in shared
  // memory, of which two workgroups then fill 149 (kBoth: 157) of 160 KB: 957 us where one
  // wave with 420 registers took 1057 (8191 tokens, 16 heads on 4, fp16).
  constexpr int kSteps = DP / 16, kFromLds = SC == kBoth ? 3 : 2, kInRegs = kSteps - kFromLds;  // of K's operands
  __shared__ Frag<T> kept[kHalf ? kWaves : 1][kHalf ? kSteps + kFromLds : 1][WAVE];
  // Names of their own: in one array the compiler takes a read of one buffer for one of the
  // other's too, and waits for the tile on its way.
  __shared__ __attribute__((aligned(16))) T qs0[QT * DP], qs1[QT * DP], gs0[QT * DP], gs1[QT * DP];
  __shared__ __attribute__((aligned(16))) float stats[2][2][QT];  // lse, delta
  __shared__ __attribute__((aligned(16))) int qd[2][QT];
  const int t = threadIdx.x, lane = t % WAVE, half = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(t / WAVE);
  const int64_t linear = xcd_order(blockIdx.x, gridDim.x);
  const int split = linear % splits;
  int64_t bc = linear / splits / k_blocks;
  // under a causal mask first, last, second, ..: the first blocks have the most queries,
  // and an XCD has a stretch of this order
  const int place = static_cast<int>(linear / splits % k_blocks);
  int j0 = (!a.causal || a.k_doc != nullptr ? tile_at(place, k_blocks, bc, false) : place % 2 == 0 ? place / 2 : k_blocks - 1 - place / 2) * kKeys;
  if (a.k_order != nullptr) j0 = ordered(a.k_order, linear / splits, k_blocks, a.B, a.Hk, bc) * kKeys;
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
  if constexpr (kHalf) {  // a lane's own operands: it reads what it wrote
#pragma unroll
    for (int x = 0; x < kSteps; ++x) kept[wave][x][lane] = vf[x];
#pragma unroll
    for (int x = 0; x < kFromLds; ++x) kept[wave][kSteps + x][lane] = kf[kInRegs + x];
  }
  // the first query that sees a key
  const int prefix = a.prefix != nullptr ? a.prefix[b] : 0;
  const int begin = !ok ? INT_MAX : !a.causal || j < prefix ? 0 : max(0, j - off);
  const int least_begin = wave_min(begin), most_begin = wave_max(begin);
  const int doc_lo = wave_min(doc), doc_hi = wave_max(doc);
  const int doc_least = doc_lo >= 0 ? doc_lo : wave_min(ok && doc >= 0 ? doc : INT_MAX);
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
  // the workgroup's part of the (head, tile) pairs: even stretches of them
  const int first_tile = min(i_begin / kDocTile, q_tiles), per_head = q_tiles - first_tile;
  const int64_t units = static_cast<int64_t>(group) * per_head;
  const int64_t unit_begin = units * split / splits, unit_end = units * (split + 1) / splits;
  int64_t unit = unit_begin;  // where the walk of the present head began
  int head = kv * group, rest = -1;
  TileWalk walk(own, lo, hi, 0, 0);
  auto enter = [&]() {  // the head that holds `unit`
    const int g = static_cast<int>(unit / per_head);
    const int64_t base = static_cast<int64_t>(g) * per_head;
    head = kv * group + g;
    walk = TileWalk(own, lo, hi, first_tile + static_cast<int>(unit - base),
                    first_tile + static_cast<int>(min(static_cast<int64_t>(per_head), unit_end - base)));
    unit = base + per_head;
  };
  auto next = [&](int& at_head) {
    if (QT < kDocTile && rest >= 0) {
      const int i = rest;
      rest = -1;
      at_head = head;
      return i;
    }
    int n = walk.next();
    while (n < 0) {
      if (unit >= unit_end) return -1;
      enter();
      n = walk.next();
    }
    if (QT < kDocTile && n * kDocTile + QT < a.Lq) rest = n * kDocTile + QT;
    at_head = head;
    return n * kDocTile;
  };
  constexpr float kWeightLift = sizeof(T) == 2 && std::is_same<T, fp16_t>::value ? 10.f : 0.f;  // see grad_scale
  float lift = 1.f;
  if constexpr (std::is_same<T, fp16_t>::value) lift = in ? a.key_lift[bc * a.Lk + j] * exp2f(-kWeightLift) : 1.f;  // the weights in dS bring theirs
  const int* d0 = a.q_doc != nullptr ? a.q_doc + static_cast<int64_t>(b) * a.Lq : nullptr;

  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int x = 0; x < DP / 32; ++x) dk[x] = zeros16(), dv[x] = zeros16();
  const Reader<T, DP> reader;
  // The scores of 32 queries pass under the weights of the 32 before, and those'
  // products under the weights of these.
  constexpr int kSub = QT / 32, kWide = DP / 32;
  auto step = [&](bool masked, int i0, float slope2, auto buf) {
    const Reader<T, DP> at = reader.fresh();
    f32x16 s[kSub], dp[kSub];
    Frag<T> p[kSub][2], ds[kSub][2], left[FINE ? kSub : 1][2];
    auto score = [&](int n, int i, const Frag<T>& f) {
      if (i == 0) s[n] = zeros16(), dp[n] = zeros16();
      if (i % 2 == 0) product(f, kf[i / 2], s[n]);
      else product(f, vf[i / 2], dp[n]);
    };
    auto score_read = [&](int n, int i) { return at.rows(i % 2 == 0 ? (buf == 0 ? qs0 : qs1) : (buf == 0 ? gs0 : gs1), 32 * n, i / 2); };
    auto output = [&](int n, int i, const Frag<T>& f) {
      if (i % 2 == 0) product(f, p[n][i / 2 / kWide], dv[i / 2 % kWide]);
      else product(f, ds[n][i / 2 / kWide], dk[i / 2 % kWide]);
      if constexpr (FINE)
        if (i % 2 == 1) product(f, left[n][i / 2 / kWide], dk[i / 2 % kWide]);
    };
    auto output_read = [&](int n, int i) { return at.columns(i % 2 == 0 ? (buf == 0 ? gs0 : gs1) : (buf == 0 ? qs0 : qs1), 32 * n + 16 * (i / 2 / kWide), i / 2 % kWide); };
    // One body for all tiles: bodies that differ by their masks would each keep the sums
    // in registers of their own.  What is not seen gets a score of -infinity, or, behind a
    // cap, its weight's bits taken away; a dP there that is not finite makes the row be
    // done again.
    uint32_t bits[kSub];
    auto mask = [&](int n) {
      bits[n] = ~0u;
      auto apply = [&](auto which) {
        Seen<decltype(which)::value, true> seen((begin == INT_MAX ? 1 << 20 : begin - i0) - 32 * n, doc, qd[buf] + 32 * n);
        if (capped(SC)) bits[n] = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (capped(SC)) bits[n] |= static_cast<uint32_t>(seen(r)) << r;
          else s[n][r] = seen(r) ? s[n][r] : -INFINITY;
        }
      };
      if (masked && own == nullptr) apply(std::integral_constant<Mask, kEnds>());
      if (masked && own != nullptr) apply(std::integral_constant<Mask, kIds>());
    };
    float4 lse, del;
    auto weight = [&](int n, int r) {  // registers r and r + 1, in their order
      // the distance |i + off - j| with queries in registers: as if the key stood at j - off
      const ScoreMap<T, SC> map(a, slope2, j - off - i0 - 32 * n);
      if (r % 4 == 0) {
        lse = *reinterpret_cast<const float4*>(&stats[buf][0][32 * n + 2 * r + 4 * half]);
        del = *reinterpret_cast<const float4*>(&stats[buf][1][32 * n + 2 * r + 4 * half]);
      }
      const float ls[2] = {r % 4 == 0 ? lse.x : lse.z, r % 4 == 0 ? lse.y : lse.w}, de[2] = {r % 4 == 0 ? del.x : del.z, r % 4 == 0 ? del.y : del.w};
      float w[2], g[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float bend;
        const float t = map(s[n][r + y], r + y, bend);
        w[y] = __builtin_amdgcn_exp2f(fmaf(t, map.factor, -ls[y]));
        if (capped(SC)) w[y] = with_bit(w[y], bits[n], r + y);
        g[y] = w[y] * (dp[n][r + y] - de[y]);
        if (capped(SC)) g[y] *= bend;
        if (std::is_same<T, fp16_t>::value) g[y] *= lift;
      }
      p[n][r / 8].set2(r % 8, w[0], w[1]);
      ds[n][r / 8].set2(r % 8, g[0], g[1]);
      if constexpr (FINE) left[n][r / 8].set2(r % 8, g[0] - to_f(ds[n][r / 8].v[r % 8]), g[1] - to_f(ds[n][r / 8].v[r % 8 + 1]));
    };
    constexpr int kA = 2 * kSteps, kB = 4 * kWide;  // products of scores and of outputs: as many
    static_assert(kA == kB && 16 % kA == 0, "pairs of registers go by products");
    constexpr int kRows = 16 / kA < 2 ? 2 : 16 / kA, kEvery = kA / (16 / kRows);  // rows at every so many products
    auto weights_beside = [&](int n, int i) {
      if (i % kEvery == 0)
#pragma unroll
        for (int r = kRows * (i / kEvery); r < kRows * (i / kEvery + 1); r += 2) weight(n, r);
    };
    if constexpr (kSub == 2) {
      piped<T, kA, 4>([&](auto i) { return score_read(0, i); }, [&](auto i, const Frag<T>& f) { score(0, i, f); });
      mask(0);
      piped<T, kA, 4>([&](auto i) { return score_read(1, i); },
                      [&](auto i, const Frag<T>& f) {
                        score(1, i, f);
                        weights_beside(0, i);
                      });
      mask(1);
      piped<T, 2 * kB, 4>([&](auto i) { return output_read(i / kB, i % kB); },
                          [&](auto i, const Frag<T>& f) {
                            output(i / kB, i % kB, f);
                            if (i < kB) weights_beside(1, i);
                          });
    } else {
      if constexpr (kHalf) {
        // Q, V, dO a step; K, Q, V, dO where K is not in registers
        constexpr int kThrees = 3 * kInRegs;
        int own_lane = lane;
        asm volatile("" : "+v"(own_lane));
        s[0] = dp[0] = zeros16();
        Frag<T> hold;
        piped<T, kThrees + 4 * kFromLds, 4>(
            [&](auto i) {
              constexpr int n = i < kThrees ? i % 3 + 1 : (i - kThrees) % 4, x = i < kThrees ? i / 3 : kInRegs + (i - kThrees) / 4;
              if constexpr (n == 0) return kept[wave][kSteps + x - kInRegs][own_lane];
              else if constexpr (n == 2) return kept[wave][x][own_lane];
              else return at.rows(n == 1 ? (buf == 0 ? qs0 : qs1) : (buf == 0 ? gs0 : gs1), 0, x);
            },
            [&](auto i, const Frag<T>& f) {
              constexpr int n = i < kThrees ? i % 3 + 1 : (i - kThrees) % 4, x = i < kThrees ? i / 3 : kInRegs + (i - kThrees) / 4;
              if constexpr (n % 2 == 0) hold = f;
              else if constexpr (n == 1) product(f, x < kInRegs ? kf[x] : hold, s[0]);
              else product(f, hold, dp[0]);
            });
      } else {
        piped<T, kA, 4>([&](auto i) { return score_read(0, i); }, [&](auto i, const Frag<T>& f) { score(0, i, f); });
      }
      mask(0);
#pragma unroll
      for (int r = 0; r < 16; r += 2) weight(0, r);
      __builtin_amdgcn_sched_barrier(0);
      piped<T, kB, 4>([&](auto i) { return output_read(0, i); }, [&](auto i, const Frag<T>& f) { output(0, i, f); });
    }
  };
  uint32_t ids = 0, stat = 0;
  DocRange range{0, 0, 0}, range_next{0, 0, 0};
  uint64_t there = 0;
  auto load = [&](int i, int h, auto buf) {
    there = first_rows(a.Lq - i);
    const int rows = min(QT, a.Lq - i);
    const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.Lq + i;
    stat = staged_word((wave == 0 ? a.lse : a.delta) + row, lane, wave < 2 ? rows : 0);  // one wave brings lse, one delta
    if (own != nullptr) {
      range_next = walk.of(i / kDocTile);
      there = range_next.there >> (i % kDocTile);
      ids = staged_word(d0 + i, t, rows);
    }
    Flight<T, DP, QT, kWaves, kHalf>::load(q_row<T>(a, b, i, h), a.qs.l, there, a.D, (buf == 0 ? qs0 : qs1), wave);
    Flight<T, DP, QT, kWaves, kHalf>::load(g_row<T>(a, b, i, h), a.gs.l, there, a.D, (buf == 0 ? gs0 : gs1), wave);
  };
  auto landed = [&](auto buf) {
    const bool here = there >> lane & 1;
    if (wave == 0 && lane < QT) stats[buf][0][lane] = here ? __uint_as_float(stat) - kWeightLift : INFINITY;
    if (wave == 1 && lane < QT) stats[buf][1][lane] = here ? __uint_as_float(stat) : 0.f;
    if (own != nullptr && t < QT) qd[buf][t] = here ? static_cast<int>(ids) : -1;
    range = range_next;
    arrived<0>();
    __syncthreads();
  };
  int h = head, h_next = head;
  int i = next(h);
  auto turn = [&](auto buf) {
    constexpr int kBuf = decltype(buf)::value;
    const int following = next(h_next);
    const DocRange present = range;
    if (following >= 0) load(following, h_next, std::integral_constant<int, 1 - kBuf>());
    if (i + QT > least_begin && (own == nullptr || (present.lo <= doc_hi && present.hi >= doc_least))) {
      const float slope2 = a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
      bool masked = i < most_begin;
      if (own != nullptr) masked = masked || !(present.one() && doc_lo == doc_hi && present.lo == doc_lo);
      step(masked, i, slope2, buf);
    }
    landed(std::integral_constant<int, 1 - kBuf>());
    i = following;
    h = h_next;
  };
  if (i >= 0) {
    load(i, h, std::integral_constant<int, 0>());
    landed(std::integral_constant<int, 0>());
    do {
      turn(std::integral_constant<int, 0>());
      if (i >= 0) turn(std::integral_constant<int, 1>());
    } while (i >= 0);
  }
  const float drop = exp2f(-kWeightLift);
  if (splits > 1) {  // joined, and looked at, by the next kernel
    const int64_t to = ((static_cast<int64_t>(b) * a.Lk + j) * a.Hk + kv) * a.D, all = static_cast<int64_t>(a.B) * a.Lk * a.Hk * a.D;
    if (in) {
      store_column<float, DP>(part + 2 * split * all + to, dk, a.D, a.scale / lift * drop);
      store_column<float, DP>(part + (2 * split + 1) * all + to, dv, a.D, drop);
    }
    return;
  }
  uint32_t again = 0;
  if (repairs<T>(a)) again = bad_columns(in && !(finite_column(dk) && finite_column(dv)));
  if (in && !(again >> (lane % 32) & 1)) {
    const int64_t out = ((static_cast<int64_t>(b) * a.Lk + j) * a.Hk + kv) * a.D;
    store_column<T, DP>(static_cast<T*>(a.dk) + out, dk, a.D, a.scale / lift * drop);
    store_column<T, DP>(static_cast<T*>(a.dv) + out, dv, a.D, drop);
  }
  for (; again != 0; again &= again - 1) dkv_row<T>(a, b, j0 + 32 * wave + __builtin_ctz(again), kv);
}

// Sums the parts of dK and dV in their order: a wave a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_dkv_kernel(AttnArgs a, int splits, int64_t rows, const float* __restrict__ part) {
  const int lane = threadIdx.x % WAVE;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / WAVE, all = rows * a.D;
  if (row >= rows) return;
  float dk[2] = {0.f, 0.f}, dv[2] = {0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s)
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (lane + 64 * x < a.D) {
        dk[x] += part[2 * s * all + row * a.D + lane + 64 * x];
        dv[x] += part[(2 * s + 1) * all + row * a.D + lane + 64 * x];
      }
  const bool fine = fabsf(dk[0]) <= FLT_MAX && fabsf(dk[1]) <= FLT_MAX && fabsf(dv[0]) <= FLT_MAX && fabsf(dv[1]) <= FLT_MAX;
  if (repairs<T>(a) && __any(!fine)) {
    const int64_t bl = row / a.Hk;
    dkv_row<T>(a, bl / a.Lk, bl % a.Lk, row % a.Hk);
    return;
  }
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (lane + 64 * x < a.D) {
      static_cast<T*>(a.dk)[row * a.D + lane + 64 * x] = from_f<T>(dk[x]);
      static_cast<T*>(a.dv)[row * a.D + lane + 64 * x] = from_f<T>(dv[x]);
    }
}

int blocks_for(int64_t items, int64_t each) {
  const int64_t n = (items + each - 1) / each;
  TORCH_CHECK(launchable(n, kThreads), "attention: too many rows");
  return static_cast<int>(n);
}

constexpr int kComputeUnits = 256;

// Calls `fn` with the padded width and what scores go through as constants.
template <typename Fn>
void with_variant(const AttnArgs& a, Fn fn) {
  auto by_score = [&](auto width) {
    const bool biased = a.slopes != nullptr || a.scale == 0.f;
    if (biased && a.softcap > 0.f) fn(width, std::integral_constant<Score, kBoth>());
    else if (biased) fn(width, std::integral_constant<Score, kBiased>());
    else if (a.softcap > 0.f) fn(width, std::integral_constant<Score, kCapped>());
    else fn(width, std::integral_constant<Score, kPlain>());
  };
  if (a.D <= 64) by_score(std::integral_constant<int, 64>());
  else by_score(std::integral_constant<int, 128>());
}

template <typename T, int DP, Score SC>
void run_forward(const AttnArgs& a, const DocRange* ranges, const torch::TensorOptions& options, hipStream_t stream) {
  if (attention_in_tiles(a)) {
    const int64_t tiles = static_cast<int64_t>(a.B) * a.H * ((a.Lq + kQueries - 1) / kQueries);
    forward_tiles_kernel<T, DP, SC><<<blocks_for(tiles, 1), kThreads, 0, stream>>>(a, ranges, (a.Lq + kQueries - 1) / kQueries);
    return;
  }
  const int rows = a.H / a.Hk * a.Lq, row_tiles = (rows + 31) / 32;
  const int64_t groups = static_cast<int64_t>(a.B) * a.Hk * row_tiles, count = static_cast<int64_t>(a.B) * a.Hk * rows;
  // some eight workgroups a CU, so that rows of uneven length even out, but 512
  // keys for each
  const int splits = std::max<int64_t>(1, std::min<int64_t>({64, (8 * kComputeUnits + groups - 1) / groups, a.Lk / 512}));
  const int each = ((a.Lk + splits - 1) / splits + 127) / 128 * 128;
  const int used = (a.Lk + each - 1) / each;
  torch::Tensor part, stats;
  if (used > 1) {
    part = torch::empty({used, count, DP}, options.dtype(at::kFloat));
    stats = torch::empty({used, count, 2}, options.dtype(at::kFloat));
  }
  float* p = used > 1 ? part.data_ptr<float>() : nullptr;
  float2* st = used > 1 ? reinterpret_cast<float2*>(stats.data_ptr<float>()) : nullptr;
  forward_split_kernel<T, DP, SC><<<blocks_for(groups * used, 1), kThreads, 0, stream>>>(a, ranges, row_tiles, used, each, p, st);
  if (used > 1) join_splits_kernel<T, DP><<<blocks_for(count, kWaves), kThreads, 0, stream>>>(a, used, count, p, st);
}

template <typename T, int DP, Score SC>
void run_backward(const AttnArgs& a, const DocRange* k_ranges, const DocRange* q_ranges, const torch::TensorOptions& options, hipStream_t stream) {
  const int q_tiles = (a.Lq + kQueries - 1) / kQueries, k_blocks = (a.Lk + kQueries - 1) / kQueries;
  const int64_t q_grid = blocks_for(static_cast<int64_t>(a.B) * a.H * q_tiles, 1);
  // Blocks of keys that do not fill the chip four times over are split over heads and
  // queries, down to eight tiles of queries, for their sums to be joined: a causal mask makes
  // their lengths uneven, and heads that share keys make them few.  Split in four where
  // eight tiles were left of 4096 tokens, 8 heads of 128: the pass 373 us, in eight 439, as
  // the join grows; parts of 64 tiles and more even out eight times over (8191 tokens, 16
  // heads on 4, 128 fp16: not split 2570, four 1735, eight 1615).
  const int64_t base = static_cast<int64_t>(a.B) * a.Hk * k_blocks;
  const int64_t tiles = static_cast<int64_t>(a.H / a.Hk) * ((a.Lq + kDocTile - 1) / kDocTile);
  const int splits = std::max<int64_t>({1, std::min<int64_t>(4 * kComputeUnits / base, tiles / 8), std::min<int64_t>(8 * kComputeUnits / base, tiles / 64)});
  const int64_t rows = static_cast<int64_t>(a.B) * a.Lk * a.Hk;
  torch::Tensor part;
  if (splits > 1) part = torch::empty({splits, 2, rows, a.D}, options.dtype(at::kFloat));
  float* p = splits > 1 ? part.data_ptr<float>() : nullptr;
  auto launch = [&](auto fine) {
    dq_tiles_kernel<T, DP, SC, decltype(fine)::value><<<q_grid, kThreads, 0, stream>>>(a, k_ranges, q_tiles);
    if constexpr (std::is_same<T, fp16_t>::value) key_lifts(a, q_ranges, stream);
    dkv_tiles_kernel<T, DP, SC, decltype(fine)::value><<<blocks_for(base * splits, 1), kThreads, 0, stream>>>(a, q_ranges, k_blocks, splits, p);
  };
  // 16-bit score gradients of rows of one tile are multiplied twice, once for what rounding took
  // from them.  Without it dQ and dK are the further off the fewer keys a row has: 1.50 times
  // as far as by the result's own rounding with 2 to 4, 1.45 with 16, 1.42 from 64 on; with it
  // 1.15 and less.  A row of one tile passes under its loads and launches either way: 64 rows
  // of 64 tokens, 12 heads of 64 fp16, dQ and dK, dV 18.8 + 17.8 us with it, 19.0 + 17.7
  // without; of 128 29.6 + 30.0 : 28.8 + 29.3.  In long rows it would be a quarter more products.
  bool done = false;
  if constexpr (sizeof(T) == 2)
    if (a.Lq <= kDocTile && a.Lk <= kDocTile) launch(std::true_type()), done = true;
  if (!done) launch(std::false_type());
  if (splits > 1) join_dkv_kernel<T><<<blocks_for(rows, kWaves), kThreads, 0, stream>>>(a, splits, rows, p);
}

}  // namespace

template <typename T>
void attention_forward(const AttnArgs& a, const DocRange* ranges, const torch::TensorOptions& options, hipStream_t stream) {
  with_variant(a, [&](auto width, auto score) {
    run_forward<T, decltype(width)::value, decltype(score)::value>(a, ranges, options, stream);
  });
}

template <typename T>
void attention_backward(const AttnArgs& a, const DocRange* k_ranges, const DocRange* q_ranges, const torch::TensorOptions& options,
                        hipStream_t stream) {
  with_variant(a, [&](auto width, auto score) {
    run_backward<T, decltype(width)::value, decltype(score)::value>(a, k_ranges, q_ranges, options, stream);
  });
}
