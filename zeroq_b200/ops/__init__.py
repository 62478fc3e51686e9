"""Hot ops: each has a PyTorch oracle (CPU) and an sm_100a kernel (CUDA)."""

from .nf4 import (NF4_CODE, FP4_CODE, QuantState, quantize_4bit, dequantize_4bit,
                  quantize_4bit_reference, dequantize_4bit_reference)
from .qlinear import Linear4bit, nf4_linear
from .gemm import gemm_bt
from .norm import add_rmsnorm, rmsnorm
from .rope import RopeScaling, apply_rope, rotary_embedding
from .activations import gelu, swiglu
from .attention import flash_attention, flash_attention_varlen
from .packed import PackedSequences
from .cross_entropy import cross_entropy
from .distill import distillation_loss
from .optim import adamw_step, lion_step

__all__ = ["NF4_CODE", "FP4_CODE", "QuantState", "quantize_4bit", "dequantize_4bit",
           "quantize_4bit_reference", "dequantize_4bit_reference", "Linear4bit", "nf4_linear",
           "gemm_bt", "add_rmsnorm", "rmsnorm", "apply_rope", "RopeScaling",
           "rotary_embedding", "gelu", "swiglu",
           "flash_attention", "flash_attention_varlen", "PackedSequences", "cross_entropy", "distillation_loss", "adamw_step", "lion_step"]
