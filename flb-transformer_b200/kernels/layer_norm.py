"""LayerNorm over the last axis on B200 (sm_100a), forward and backward.

    layer_norm(x, weight=None, bias=None, eps=1e-5, keep8=False) -> y
    layer_norm_int8(x, weight=None, bias=None, eps=1e-5) -> Int8Rows
    FusedLayerNorm(dim)                                             nn.LayerNorm that calls it

    h = (x - mean) / sqrt(var + eps),  y = h * weight + bias

x: float32, float16 or bfloat16, [..., D] with D <= 32768 (16384 where a gradient is wanted). weight and
bias: float32 or x's type, [D], or [G, D] for x [G, ..., D]: one weight for each index of x's first
axis (at most 65535 of them; a vmap over weights makes such groups). y has x's type, also under autocast,
where nn.LayerNorm's is float32. Statistics and the gradient's sums are in float32: a row whose sum overflows
there is NaN, and where its squares do, h is zero. The gradient of the weight is summed in a fixed order. With
keep8 the backward reads h from 8 bits (kernels.kept8's kept form) instead of x from its own: about half the
memory kept, and the same y.

The kernels are in libflb_b200.so (flb_layer_norm_fwd, flb_layer_norm_bwd), called through flb_ops;
CUDA tensors only.
"""
from __future__ import annotations

import torch
import torch.nn as nn

import flb_native  # noqa: F401  (loads libflb_b200.so, or says that it is missing)
import flb_ops
from ._rows import backward_of, no_transforms, to_front, transforms_active
from .int8_linear import Int8Rows

__all__ = ["layer_norm", "layer_norm_int8", "FusedLayerNorm"]


class _LayerNormFunc(torch.autograd.Function):
    """layer_norm under torch.func transforms: what the backward reads are outputs of the forward."""

    @staticmethod
    def forward(x, weight, bias, eps, keep8):
        return tuple(t for t in flb_ops.norm_forward(x, weight, bias, eps, keep8, True) if t is not None)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, weight, bias, _, ctx.keep8 = inputs
        # 1/sigma is not marked: with keep8 it alone tells the levels of torch.func that what the backward reads depends on x
        ctx.mark_non_differentiable(*output[2:])
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(None if ctx.keep8 else x, weight, bias, *output[1:])

    @staticmethod
    def backward(ctx, dy, *_):
        x, weight, bias, rstd, *kept = ctx.saved_tensors
        mean, codes, exps = (None, *kept) if ctx.keep8 else (kept[0], None, None)
        dx, *params = backward_of(flb_ops.norm_backward, x, rstd, mean, codes, exps, weight, bias, dy, True)
        dw = params.pop(0) if weight is not None else None
        return dx, dw, params.pop(0) if bias is not None else None, None, None

    @staticmethod
    def vmap(info, in_dims, x, weight, bias, eps, keep8):
        # samples become groups, each with its own weight, or with groups of its own under it
        size = info.batch_size
        xd, wd, bd = in_dims[:3]
        x = to_front(x, xd, size)
        inner = x.shape
        like, ld = (weight, wd) if weight is not None else (bias, bd)
        grouped = like is not None and like.ndim - (ld is not None) == 2
        if wd is not None or bd is not None or grouped:
            weight, bias = (None if t is None else to_front(t, d, size) for t, d in ((weight, wd), (bias, bd)))
            if grouped:
                weight, bias = (None if t is None else t.reshape(-1, t.shape[-1]) for t in (weight, bias))
                x = x.reshape(-1, *x.shape[2:])
        out = _LayerNormFunc.apply(x, weight, bias, eps, keep8)
        return (out[0].reshape(inner), *out[1:]), (0, *(None,) * (len(out) - 1))


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, keep8: bool = False) -> torch.Tensor:
    """LayerNorm of x's last axis (see the module's text). Differentiable once; torch.vmap is supported."""
    if transforms_active():
        return _LayerNormFunc.apply(x, weight, bias, float(eps), bool(keep8))[0]
    return flb_ops.layer_norm(x, weight, bias, eps, keep8)


def layer_norm_int8(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                    eps: float = 1e-5) -> Int8Rows:
    """The rows of layer_norm's output, before their rounding to x's type, as 8-bit integers: the input that
    int8_linear reads, in one pass over x. No gradient."""
    no_transforms("layer_norm_int8")
    return Int8Rows(*flb_ops.layer_norm_int8(x, weight, bias, eps), x.dtype)


class FusedLayerNorm(nn.LayerNorm):
    """nn.LayerNorm over one last axis with the same parameters, whose forward is layer_norm. keep8 as
    there."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 keep8: bool = False, device=None, dtype=None):
        super().__init__(dim, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("FusedLayerNorm normalises one axis")
        self.keep8 = keep8

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1:] != torch.Size(self.normalized_shape):
            raise ValueError(f"x of shape {tuple(x.shape)} for a norm over {self.normalized_shape[0]} elements")
        return layer_norm(x, self.weight, self.bias, self.eps, self.keep8)
