// Between the entry points of attention and its kernels, which are compiled one
// element type to a source file.
#pragma once

#include <torch/extension.h>

#include "attention_tile.h"

template <typename T>
void attention_forward(const AttnArgs& a, const DocRange* ranges, const torch::TensorOptions& options, hipStream_t stream);

// `a.delta` (and `a.grad_top`, zeroed, for fp16) are written here.
template <typename T>
void attention_backward(const AttnArgs& a, const DocRange* k_ranges, const DocRange* q_ranges, const torch::TensorOptions& options,
                        hipStream_t stream);
