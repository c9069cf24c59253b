// The attention kernels for fp32.
#include "attention_kernels.h"

template void attention_forward<float>(const AttnArgs&, const DocRange*, const torch::TensorOptions&, hipStream_t);
template void attention_backward<float>(const AttnArgs&, const DocRange*, const DocRange*, const torch::TensorOptions&, hipStream_t);
