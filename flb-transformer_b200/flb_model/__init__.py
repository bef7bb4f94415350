"""FLB-Transformer on this package's operators: the model (same math and parameter names as
the reference's models/FLB_Model.py) and decode loops for it."""
from .model import FLBAttentionLayer, FLBBlock, FLBTransformer, FLB_DEPENDENCIES
from .decode import greedy_decode, sample_decode

__all__ = ["FLBAttentionLayer", "FLBBlock", "FLBTransformer", "FLB_DEPENDENCIES",
           "greedy_decode", "sample_decode"]
