"""B200-native fused 4-bit dequantise-and-multiply behind a Jenks-quantized Linear, and linears in 8-bit integers.

Public surface:
    JenksQuantLinear, quantize_module   -- drop-in for the reference's QuantLinear
    QuantSpec, PackedWeight, pack_weight -- packed formats and the host packer
    ops.linear / ops.dequantize / ops.fwht_block / ops.GroupedGemv -- kernels
    KVCache                             -- 8-bit key/value cache: append, read, attend
    ops.quantize_rows                   -- activations in 8-bit integers by token, which ops.linear takes too
    ops.residual_norm                   -- the norms around a block with its gate and residual sum, in 16 or 8 bits
    ops.token_logprobs                  -- log probabilities of tokens, entropy, strongest alternatives
All compute goes through libjq.so (include/jq.h); nothing falls back to CPU.
"""
from .spec import QuantSpec, algorithmic_bytes  # noqa: F401
from .pack import PackedWeight, pack_weight  # noqa: F401
from . import ops  # noqa: F401
from .linear import JenksQuantLinear, quantize_module  # noqa: F401
from .conv import JenksQuantConv2d  # noqa: F401
from .cache import KVCache  # noqa: F401

__all__ = ["QuantSpec", "PackedWeight", "pack_weight", "ops", "JenksQuantLinear", "JenksQuantConv2d", "quantize_module", "KVCache",
           "algorithmic_bytes"]
