"""Operators on B200: additive attention (the B200 build of FLB-Transformer's kernels package), LayerNorm,
the sigmoid gate, and activations kept in 8 bits."""
from .additive_attention import FusedAdditiveAttentionFunc, fused_additive_attention
from .kept8 import Packed8, pack8, sigmoid_gate, unpack8
from .layer_norm import FusedLayerNorm, layer_norm

__all__ = ["FusedAdditiveAttentionFunc", "fused_additive_attention", "FusedLayerNorm", "layer_norm", "Packed8",
           "pack8", "unpack8", "sigmoid_gate"]
