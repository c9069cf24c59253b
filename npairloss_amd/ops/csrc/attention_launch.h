// Between the entry points of attention and its kernels, which are compiled one
// element type to a source file.
#pragma once

#include <torch/extension.h>

#include "attention_tile.h"

// Whether queries go in tiles of 128 or by 32 with their keys in stretches.  Tiles use every
// key tile four times as often but have nothing to share out over keys: they take rows that
// fill the chip, and short keys, where the stretches' join is the longer part.  12 heads of 64
// bf16, batch x queries, tiles against stretches in us: 256 keys 1x128 11 : 13, 64x8 15 : 16;
// 1024 keys 4x128 25 : 22, 8x128 25 : 27, 64x32 36 : 57; 4096 keys 8x128 80 : 66,
// 16x128 83 : 93, 16x32 74 : 52, 64x32 147 : 176, 64x64 153 : 260.
inline bool attention_in_tiles(const AttnArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.H / a.Hk) * a.Lq, groups = static_cast<int64_t>(a.B) * a.Hk * ((rows + 31) / 32);
  return a.Lk <= 384 || (a.Lq >= 32 && groups >= 512);
}

template <typename T>
void attention_forward(const AttnArgs& a, const DocRange* ranges, const torch::TensorOptions& options, hipStream_t stream);

// `a.key_lift` from `a.row_top` and `a.block_top`.
void key_lifts(const AttnArgs& a, const DocRange* q_ranges, hipStream_t stream);

// `a.delta` (and for fp16 `a.row_top`, `a.block_top` and `a.key_lift`) are written here.
template <typename T>
void attention_backward(const AttnArgs& a, const DocRange* k_ranges, const DocRange* q_ranges, const torch::TensorOptions& options,
                        hipStream_t stream);
