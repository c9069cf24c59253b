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

#include <utility>

using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned int;

template <typename T>
struct Frag {  // eight k of one row or column
  using V = __attribute__((ext_vector_type(8))) T;
  V v;
  DEVINL void set2(int i, float x, float y) {  // one conversion for two
    using F2 = __attribute__((ext_vector_type(2))) float;
    using T2 = __attribute__((ext_vector_type(2))) T;
    const T2 t = __builtin_convertvector((F2{x, y}), T2);
    v[i] = t[0];
    v[i + 1] = t[1];
  }
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

// N products in a row, each with an operand from shared memory: `read(i)` brings it,
// AHEAD of them before the first `use(i, operand)` and one more behind each, so that a
// read's latency passes under products and under what else `use` does.  The compiler
// left alone waits for every read in front of its product; the barriers hold the
// order as it is written.
template <typename Fn, int... I>
DEVINL void each(std::integer_sequence<int, I...>, Fn fn) {
  (fn(std::integral_constant<int, I>()), ...);
}

template <typename T, int N, int AHEAD, typename Read, typename Use>
DEVINL void piped(Read read, Use use) {
  Frag<T> f[AHEAD];
  each(std::make_integer_sequence<int, AHEAD>(), [&](auto i) { f[i] = read(i); });
  __builtin_amdgcn_sched_barrier(0);
  each(std::make_integer_sequence<int, N>(), [&](auto i) {
    use(i, f[i % AHEAD]);
    if constexpr (i + AHEAD < N) f[i % AHEAD] = read(std::integral_constant<int, i + AHEAD>());
    __builtin_amdgcn_sched_barrier(0);
  });
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

};

// A wave's way of reading operands from a tile.  A lane's places differ from its
// first by constants, under XOR (the swizzle is linear in the bits of the row) and in
// the offset: two registers hold all of them, and `fresh` keeps the compiler from
// holding every one over the loop instead.
template <typename T, int DP>
struct Reader {
  using Tl = Tile<T, DP>;
  static constexpr bool kWide = sizeof(T) == 4;
  int row_at;  // elements: row lane % 32, its eight k of step 0
  int col_at;  // elements: a lane's place for columns, x = 0, its first row

  DEVINL Reader() {
    const int lane = threadIdx.x % WAVE, half = lane / 32;
    row_at = Tl::chunk_at(lane % 32, (kWide ? 2 : 1) * half) * Tl::kPer;
    if constexpr (kWide) {
      col_at = Tl::chunk_at(4 * half, lane % 32 / 4) * 4 + lane % 4;
    } else {
      const int j = lane % 16, col = lane / 16 % 2 * 16 + j % 4 * 4;
      col_at = Tl::chunk_at(4 * half + j / 4, col / 8) * 8 + col % 8;
    }
  }

  DEVINL Reader fresh() const {
    Reader r = *this;
    asm volatile("" : "+v"(r.row_at), "+v"(r.col_at));
    return r;
  }

  DEVINL void move(int rows) {  // by a multiple of 16
    row_at += rows * DP;
    col_at += rows * DP;
  }

  // Row row0 + lane % 32 (row0 a multiple of 16), k = 16 step + 8 half ...: an
  // operand as it lies.
  DEVINL Frag<T> rows(const T* tile, int row0, int step) const {
    Frag<T> f;
    u32x4* out = reinterpret_cast<u32x4*>(&f.v);
    out[0] = *reinterpret_cast<const u32x4*>(tile + row0 * DP + (row_at ^ 16 * step));
    if constexpr (kWide) out[1] = *reinterpret_cast<const u32x4*>(tile + row0 * DP + (row_at ^ 16 * step ^ 4));
    return f;
  }

  // Column 32 x + lane % 32 of rows row0 .. row0 + 15 (row0 a multiple of 16), in
  // the order of results: an operand transposed.
  DEVINL Frag<T> columns(const T* tile, int row0, int x) const {
    Frag<T> f;
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = 8 * (i / 4) + i % 4;
        f.v[i] = tile[(row0 + row) * DP + (col_at ^ 32 * x ^ Tl::swizzle(row) * 4)];
      }
    } else {
      s16x4* out = reinterpret_cast<s16x4*>(&f.v);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        out[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(const_cast<T*>(tile + (row0 + 8 * i) * DP + (col_at ^ 32 * x ^ Tl::swizzle(8 * i) * 8))));
    }
    return f;
  }
};

// Global rows straight to a tile in shared memory, 16 bytes a lane, by WAVES waves.
// A load writes its lanes' chunks one behind another, so each lane asks for the chunk
// that belongs at its place: within a tile rows n steps apart differ by a constant in
// the swizzle.  Rows without their bit in `there` and chunks behind the width come
// as zeros (an offset beyond the buffer's end reads as zero).  Nothing waits here:
// `arrived` does, and the compiler knows of no dependence.
// FRESH: a lane's offsets are worked out each time, not held over a loop.
template <typename T, int DP, int ROWS, int WAVES, bool FRESH = false>
struct Flight {
  using Tl = Tile<T, DP>;
  static constexpr int kStep = WAVES * WAVE / Tl::kChunks;  // rows of one load of all waves
  static constexpr int kLoads = ROWS / kStep;
  static_assert(ROWS % kStep == 0 && (kStep & (kStep - 1)) == 0, "waves share the rows evenly");

  static DEVINL void load(const T* base, int64_t row_stride, uint64_t there, int D, T* tile, int wave) {
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, 0x7FFFFFFF, 0x00020000);
    const int stride = static_cast<int>(row_stride) * static_cast<int>(sizeof(T));
    int place = wave * WAVE + threadIdx.x % WAVE;
    if (FRESH) asm volatile("" : "+v"(place));
    const int row = place / Tl::kChunks, c = place % Tl::kChunks ^ Tl::swizzle(row);
    const int at = row * stride;
    // full tiles of full rows need no look at every row
    const bool full = D == DP && (ROWS == 32 ? static_cast<uint32_t>(there) == ~0u : there == ~uint64_t{0});
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int chunk = c ^ Tl::swizzle(n * kStep);
      int from = at + chunk * 16;
      if (!full) from = (there >> (row + n * kStep) & 1) && chunk * Tl::kPer < D ? from : -1;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)(tile + (n * WAVES + wave) * WAVE * Tl::kPer), 16, from, n * kStep * stride, 0, 0);
    }
  }
};

// All but the last `N` loads of this wave are in shared memory.  The builtin and not asm:
// the compiler then knows that loads into registers have arrived, too, and has no wait
// of its own for them among the products of a loop.
template <int N>
DEVINL void arrived() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);  // vmcnt N, the others as they are
  asm volatile("" ::: "memory");
}
// All reads of shared memory of this wave are in registers.
DEVINL void read_out() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The tile of a head that place `i` of `n` takes.  Under a causal mask the last tiles
// are the longest and go first.  Otherwise heads begin at different tiles: workgroups
// that are a multiple of an XCD's CUs apart start on the same CU, and would all be
// the same tile of several heads, all long or all short.
DEVINL int tile_at(int i, int n, int64_t head, bool longest_first) {
  if (longest_first) return n - 1 - i;
  const uint32_t turn = static_cast<uint32_t>((static_cast<uint64_t>(static_cast<uint32_t>(head) * 0x9E3779B9u) * n) >> 32);
  return (i + turn) % n;
}

// The same with blocks of rows in an order of their own, [B, n], longest first: an XCD's
// heads, which neighbour in `place`, go through it side by side.  Sets `head`.
DEVINL int ordered(const int* order, int64_t place, int n, int B, int heads, int64_t& head) {
  const int64_t all = static_cast<int64_t>(B) * heads, side = all % 8 == 0 ? all / 8 : 1;
  const int64_t first = place / (side * n), in = place % (side * n);
  head = first * side + in % side;
  return order[head / heads * n + in / side];
}

// One word a thread, the first `n` of them, on the same way.
DEVINL uint32_t staged_word(const void* base, int t, int n) {
  auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7FFFFFFF, 0x00020000);
  return __builtin_amdgcn_raw_buffer_load_b32(rsrc, t < n ? 4 * t : -1, 0, 0);
}

// The first `n` of 64 rows, as bits.
DEVINL uint64_t first_rows(int n) { return n >= 64 ? ~uint64_t{0} : n <= 0 ? 0 : (uint64_t{1} << n) - 1; }

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

// The ids of 64 rows (of one batch row): the least and largest that are not
// negative (an empty range without any), and which rows have one.
struct DocRange {
  int lo, hi;
  uint64_t there;
  DEVINL bool one() const { return lo == hi && there == ~uint64_t{0}; }
};
constexpr int kDocTile = 64;

// Which tiles of 64 rows an interval of ids may meet: 64 of them at a time, a lane
// holds one's ids.
struct TileWalk {
  const DocRange* ranges;  // or null: all
  int lo, hi;              // ids on the other side
  int next_base, end;      // tiles [.., end)
  uint64_t bits;
  int base;
  DocRange mine;           // of tile base + lane

  DEVINL TileWalk(const DocRange* r, int lo_, int hi_, int begin, int end_)
      : ranges(r), lo(lo_), hi(hi_), next_base(begin), end(end_), bits(0), base(begin), mine{0, 0, 0} {}

  // The next tile, or -1.  All lanes of the wave together.
  DEVINL int next() {
    while (bits == 0) {
      if (next_base >= end) return -1;
      base = next_base;
      next_base += 64;
      const int t = base + threadIdx.x % WAVE;
      bool meets = t < end;
      if (ranges != nullptr && meets) {
        mine = ranges[t];
        meets = mine.lo <= hi && mine.hi >= lo;
      }
      bits = __ballot(meets);
    }
    const int t = base + __builtin_ctzll(bits);
    bits &= bits - 1;
    return t;
  }

  // The ids of a tile that next() gave since it last took 64.
  DEVINL DocRange of(int tile) const {
    const int lane = tile - base;
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(mine.there), lane);
    const uint32_t high = __builtin_amdgcn_readlane(static_cast<uint32_t>(mine.there >> 32), lane);
    return DocRange{__builtin_amdgcn_readlane(mine.lo, lane), __builtin_amdgcn_readlane(mine.hi, lane),
                    static_cast<uint64_t>(high) << 32 | low};
  }
};
