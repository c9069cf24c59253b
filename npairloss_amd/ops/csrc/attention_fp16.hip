// The attention kernels for fp16.
#include "attention_kernels.h"

template void attention_forward<fp16_t>(const AttnArgs&, const DocRange*, const torch::TensorOptions&, hipStream_t);
template void attention_backward<fp16_t>(const AttnArgs&, const DocRange*, const DocRange*, const torch::TensorOptions&, hipStream_t);
