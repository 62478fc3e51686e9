"""Hot ops: each has a PyTorch oracle (CPU) and an sm_100a kernel (CUDA)."""

from .nf4 import (NF4_CODE, FP4_CODE, QuantState, quantize_4bit, dequantize_4bit,
                  quantize_4bit_reference, dequantize_4bit_reference)
from .qlinear import Linear4bit, nf4_linear
from .gemm import gemm_bt
from .norm import add_layer_norm, add_rmsnorm, layer_norm, rmsnorm
from .rope import RopeScaling, apply_rope, rotary_embedding
from .activations import gelu, swiglu
from .attention import flash_attention, flash_attention_varlen
from .packed import PackedSequences
from .cross_entropy import cross_entropy
from .distill import distillation_loss
from .embedding import embedding
from .act8 import Activation8, checkpoint_8bit, dequantize_activation, quantize_activation
from .logprobs import TokenLogprobs, token_logprobs
from .optim import adamw_step, lion_step

__all__ = ["NF4_CODE", "FP4_CODE", "QuantState", "quantize_4bit", "dequantize_4bit",
           "quantize_4bit_reference", "dequantize_4bit_reference", "Linear4bit", "nf4_linear",
           "gemm_bt", "add_rmsnorm", "rmsnorm", "apply_rope", "RopeScaling",
           "rotary_embedding", "gelu", "swiglu",
           "flash_attention", "flash_attention_varlen", "PackedSequences", "cross_entropy", "distillation_loss",
           "embedding", "layer_norm", "add_layer_norm", "Activation8", "quantize_activation",
           "dequantize_activation", "checkpoint_8bit", "TokenLogprobs", "token_logprobs", "adamw_step", "lion_step"]
