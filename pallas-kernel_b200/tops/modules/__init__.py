"""Modules of the GLA layer around the chunked op (reference tops/modules)."""
from .fused_norm_gate import FusedRMSNormGated, fused_rms_norm_gated
from .convolution import ShortConvolution, causal_conv1d, causal_conv1d_step
from .gate import gate_logsigmoid
from .layernorm import RMSNorm
from .qk_norm import qk_norm_rotary, rotary_tables

__all__ = ["FusedRMSNormGated", "fused_rms_norm_gated", "gate_logsigmoid", "RMSNorm", "ShortConvolution",
           "causal_conv1d", "causal_conv1d_step", "qk_norm_rotary", "rotary_tables"]
