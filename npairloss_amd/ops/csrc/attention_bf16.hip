// The attention kernels for bf16.
#include "attention_kernels.h"

template void attention_forward<bf16_t>(const AttnArgs&, const DocRange*, const torch::TensorOptions&, hipStream_t);
template void attention_backward<bf16_t>(const AttnArgs&, const DocRange*, const DocRange*, const torch::TensorOptions&, hipStream_t);
