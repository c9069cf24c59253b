// Tiles of the attention kernels: rows of K, V, Q or dO in shared memory, read as
// operands of the 32x32 matrix instructions (gfx950).
//
// A product C[32 x 32] += A[32 x 16] B[16 x 32] gives lane l row l % 32 of A and
// column l % 32 of B, eight consecutive k each (half h = l / 32 takes the other
// eight), and sixteen results of column l % 32:  row 8 (r / 4) + 4 h + r % 4.
// The order of k is free as long as A and B agree, and that is used twice:
//
//  * results of one product are operands of the next without leaving their lane.
//    Registers 8 t .. 8 t + 7 of C hold rows 16 t + 4 h + {0..3} and
//    16 t + 8 + 4 h + {0..3}; taken as eight k of B they need A's k in that order,
//    which two 4 x 16 transposing reads of shared memory give (16-bit types), or
//    eight single reads (fp32);
//  * fp32 runs as eight products of k = 2, one for each of a lane's eight values.
//
// Shared memory holds rows of DP elements in chunks of 16 bytes; chunk c of row r
// lies at c ^ swizzle(r).  Sixteen rows at one chunk, as the row reads touch
// them, and four rows at four chunks, as the transposing ones do, then lie in
// different banks.
#pragma once

#include "attention.h"

using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned int;

template <typename T> struct Frag;  // eight k of one row or column
template <> struct Frag<bf16_t> {
  using V = __attribute__((ext_vector_type(8))) bf16_t;
  V v;
  DEVINL void set(int i, float x) { v[i] = static_cast<bf16_t>(x); }
};
template <> struct Frag<fp16_t> {
  using V = __attribute__((ext_vector_type(8))) fp16_t;
  V v;
  DEVINL void set(int i, float x) { v[i] = static_cast<fp16_t>(x); }
};
template <> struct Frag<float> {
  using V = __attribute__((ext_vector_type(8))) float;
  V v;
  DEVINL void set(int i, float x) { v[i] = x; }
};

DEVINL void product(const Frag<bf16_t>& a, const Frag<bf16_t>& b, f32x16& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
DEVINL void product(const Frag<fp16_t>& a, const Frag<fp16_t>& b, f32x16& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.v, b.v, c, 0, 0, 0);
}
DEVINL void product(const Frag<float>& a, const Frag<float>& b, f32x16& c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i], b.v[i], c, 0, 0, 0);
}

DEVINL f32x16 zeros16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// The row (of 32) that result register r of a half belongs to.
DEVINL constexpr int result_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

template <typename T, int DP>
struct Tile {
  static constexpr int kPer = 16 / sizeof(T);       // elements of a chunk
  static constexpr int kChunks = DP / kPer;         // of a row: 8, 16 or 32
  static DEVINL int swizzle(int row) {
    return kChunks == 8 ? 4 * ((row >> 1) & 1) + ((row >> 2) & 3) : 4 * (row & 3) + ((row >> 2) & 3);
  }
  static DEVINL int chunk_at(int row, int c) { return row * kChunks + (c ^ swizzle(row)); }

  // Row row0 + lane % 32, k = 16 step + 8 half ...: an operand as it lies.
  static DEVINL Frag<T> rows(const T* tile, int row0, int step) {
    const int lane = threadIdx.x % WAVE, row = row0 + lane % 32, half = lane / 32;
    Frag<T> f;
    const u32x4* p = reinterpret_cast<const u32x4*>(tile);
    u32x4* out = reinterpret_cast<u32x4*>(&f.v);
    if constexpr (sizeof(T) == 2) {
      out[0] = p[chunk_at(row, 2 * step + half)];
    } else {
      out[0] = p[chunk_at(row, 4 * step + 2 * half)];
      out[1] = p[chunk_at(row, 4 * step + 2 * half + 1)];
    }
    return f;
  }

  // Column d0 + lane % 32 of rows row0 .. row0 + 15, in the order of results:
  // an operand transposed.
  static DEVINL Frag<T> columns(const T* tile, int row0, int d0) {
    const int lane = threadIdx.x % WAVE, half = lane / 32;
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
      const int j = lane % 16;
      const int col = d0 + (lane / 16) % 2 * 16 + j % 4 * 4;
      s16x4* out = reinterpret_cast<s16x4*>(&f.v);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = row0 + 8 * x + 4 * half + j / 4;
        const T* p = tile + chunk_at(row, col / 8) * 8 + col % 8;
        out[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(const_cast<T*>(p)));
      }
    } else {
      const int col = d0 + lane % 32;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = row0 + 8 * (i / 4) + 4 * half + i % 4;
        f.v[i] = tile[chunk_at(row, col / 4) * 4 + col % 4];
      }
    }
    return f;
  }
};

// Global rows on their way to shared memory, in registers: NT threads, ROWS rows.
// Rows from `count` on, chunks behind the width and rows whose id is negative
// come as zeros (an offset beyond the buffer's end reads as zero).
template <typename T, int DP, int ROWS, int NT>
struct Staged {
  using Tl = Tile<T, DP>;
  static constexpr int kEach = ROWS * Tl::kChunks / NT;
  static_assert(ROWS * Tl::kChunks % NT == 0, "threads share the chunks evenly");
  u32x4 r[kEach];

  DEVINL void load(const T* base, int64_t row_stride, int count, int D, const int* doc, int t) {
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, 0x7FFFFFFF, 0x00020000);
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const int i = t + n * NT, row = i / Tl::kChunks, c = i % Tl::kChunks;
      bool ok = row < count && c * Tl::kPer < D;
      if (doc != nullptr && ok) ok = doc[row] >= 0;
      const int at = static_cast<int>(row * row_stride + c * Tl::kPer) * static_cast<int>(sizeof(T));
      r[n] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, ok ? at : -1, 0, 0);
    }
  }

  DEVINL void store(T* tile, int t) const {
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const int i = t + n * NT, row = i / Tl::kChunks, c = i % Tl::kChunks;
      reinterpret_cast<u32x4*>(tile)[Tl::chunk_at(row, c)] = r[n];
    }
  }
};

// Row `row` (per lane) of q or dO straight into operands: k = 16 step + 8 half ...
template <typename T, int DP>
DEVINL void load_operands(const T* row, bool ok, int D, Frag<T> (&f)[DP / 16]) {
  const int half = threadIdx.x % WAVE / 32;
#pragma unroll
  for (int step = 0; step < DP / 16; ++step) {
    const int d = 16 * step + 8 * half;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[step].v[i] = static_cast<T>(0.f);
    if (ok && d < D) f[step].v = *reinterpret_cast<const typename Frag<T>::V*>(row + d);
  }
}

DEVINL float other_half(float v) { return __shfl_xor(v, 32, WAVE); }

DEVINL int wave_min(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off, WAVE));
  return __builtin_amdgcn_readfirstlane(v);
}
DEVINL int wave_max(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, WAVE));
  return __builtin_amdgcn_readfirstlane(v);
}

// Neighbouring workgroups run on different XCDs, each with an L2 of its own:
// gives each XCD a contiguous stretch of the work instead.
DEVINL int64_t xcd_order(int64_t i, int64_t n) {
  const int64_t each = n / 8, more = n % 8, x = i % 8;
  return x * each + min(x, more) + i / 8;
}

// The ids of 64 rows (of one batch row): {least, largest, 1 if all 64 are one
// id >= 0}; negative ids do not count, and without any the range is empty.
struct DocRange { int lo, hi, one, pad; };
constexpr int kDocTile = 64;

// Which tiles of 64 rows an interval of ids may meet: 64 of them at a time.
struct TileWalk {
  const DocRange* ranges;  // or null: all
  int lo, hi;              // ids on the other side
  int next_base, end;      // tiles [.., end)
  uint64_t bits;
  int base;

  DEVINL TileWalk(const DocRange* r, int lo_, int hi_, int begin, int end_)
      : ranges(r), lo(lo_), hi(hi_), next_base(begin), end(end_), bits(0), base(begin) {}

  // The next tile, or -1.  All lanes of the wave together.
  DEVINL int next() {
    while (bits == 0) {
      if (next_base >= end) return -1;
      base = next_base;
      next_base += 64;
      const int t = base + threadIdx.x % WAVE;
      bool meets = t < end;
      if (ranges != nullptr && meets) meets = ranges[t].lo <= hi && ranges[t].hi >= lo;
      bits = __ballot(meets);
    }
    const int t = base + __builtin_ctzll(bits);
    bits &= bits - 1;
    return t;
  }
};
