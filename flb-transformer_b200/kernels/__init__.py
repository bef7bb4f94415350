"""Operators on B200: additive attention (the B200 build of FLB-Transformer's kernels package), LayerNorm,
the sigmoid gate, activations kept in 8 bits, and linear maps in 8-bit integers."""
from .additive_attention import FusedAdditiveAttentionFunc, fused_additive_attention
from .int8_linear import Int8Linear, Int8Rows, int8_linear, quantize_int8
from .kept8 import Packed8, pack8, sigmoid_gate, unpack8
from .layer_norm import FusedLayerNorm, layer_norm, layer_norm_int8

__all__ = ["FusedAdditiveAttentionFunc", "fused_additive_attention", "FusedLayerNorm", "layer_norm",
           "layer_norm_int8", "Packed8", "pack8", "unpack8", "sigmoid_gate", "Int8Linear", "Int8Rows",
           "int8_linear", "quantize_int8"]
