// Between the entry points of attention and its kernels, which are compiled one
// element type to a source file.
#pragma once

#include <torch/extension.h>

#include "attention_tile.h"

// Tiles of queries where they fill the chip and their 128 rows are mostly there; 32
// rows and stretches of keys where not.
inline bool attention_in_tiles(const AttnArgs& a) {
  constexpr int kRows = 2 * kDocTile, kComputeUnits = 256;
  return a.Lq >= 64 && static_cast<int64_t>(a.B) * a.H * ((a.Lq + kRows - 1) / kRows) >= kComputeUnits;
}

template <typename T>
void attention_forward(const AttnArgs& a, const DocRange* ranges, const torch::TensorOptions& options, hipStream_t stream);

// `a.delta` (and `a.grad_top`, zeroed, for fp16) are written here.
template <typename T>
void attention_backward(const AttnArgs& a, const DocRange* k_ranges, const DocRange* q_ranges, const torch::TensorOptions& options,
                        hipStream_t stream);
