from .npair_loss import NPairMultiClassLoss, NPairLossOutput
from .l2norm import L2Normalize, l2_normalize
from .rmsnorm import RMSNorm, rms_norm, rms_norm_fp8
from .rotary_positions import rotary, rotary_frequencies
from .masked_attention import attention
from .adamw import adamw_state, adamw_step

__all__ = ["NPairMultiClassLoss", "NPairLossOutput", "L2Normalize", "l2_normalize",
           "RMSNorm", "rms_norm", "rms_norm_fp8", "rotary", "rotary_frequencies",
           "attention", "adamw_state", "adamw_step"]
