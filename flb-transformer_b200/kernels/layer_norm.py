"""LayerNorm over the last axis on B200 (sm_100a), forward and backward.

    layer_norm(x, weight=None, bias=None, eps=1e-5, keep8=False) -> y
    FusedLayerNorm(dim)                                             nn.LayerNorm that calls it

    h = (x - mean) / sqrt(var + eps),  y = h * weight + bias

x: float32, float16 or bfloat16, [..., D] with D <= 32768 (16384 where a gradient is wanted). weight and
bias: float32 or x's type, [D], or [G, D] for x [G, ..., D]: one weight for each index of x's first
axis. y has x's type; statistics and the gradient's sums are in float32, and the gradient of the weight
is summed in a fixed order. With keep8 the backward reads h from 8 bits (kernels.kept8's kept form) instead
of x from its own: about half the memory kept, and the same y.

The kernels are in libflb_b200.so (flb_layer_norm_fwd, flb_layer_norm_bwd); CUDA tensors only.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

import flb_native as nat
from ._rows import as_rows, dtype_of, on_device_of, plain, same_device, to_front, transforms_active
from .kept8 import kept_buffers

__all__ = ["layer_norm", "FusedLayerNorm"]


def _check(x, weight, bias):
    """(dtype code, weight dtype code, groups, rows a group, D)"""
    dt = dtype_of(x, "x")
    same_device(x, weight, bias)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have a last axis of at least one element, not shape {tuple(x.shape)}")
    D, G, wdt = x.shape[-1], 1, dt
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        wdt = dtype_of(t, name)
        if wdt != nat.F32 and wdt != dt:
            raise TypeError(f"{name} must be float32 or {x.dtype}, not {t.dtype}")
        if t.shape[-1:] != x.shape[-1:] or t.ndim > 2 or (t.ndim == 2 and (x.ndim < 2 or t.shape[0] != x.shape[0])):
            raise ValueError(f"{name} of shape {tuple(t.shape)} for x of shape {tuple(x.shape)}: "
                             "[D], or [G, D] with G x's first axis")
        if t.ndim == 2:
            G = t.shape[0]
    if weight is not None and bias is not None and (weight.shape != bias.shape or weight.dtype != bias.dtype):
        raise ValueError("weight and bias differ in shape or type")
    rows = x.numel() // D
    return dt, wdt, G, rows // G if G else 0, D


def _forward(x, weight, bias, eps, keep8, stats):
    """y and (mean, rstd, codes, exps), each None where the backward would not read it."""
    dt, wdt, G, R, D = _check(x, weight, bias)
    if stats and D > 16384:
        raise RuntimeError("layer_norm: the gradient of rows wider than 16384 is not supported")
    x, ldx = as_rows(x)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = codes = exps = None
    if stats:
        rstd = torch.empty(G * R, dtype=torch.float32, device=x.device)
        if keep8:
            codes, exps = kept_buffers(G * R, D, x.device)
        else:
            mean = torch.empty_like(rstd)
    with on_device_of(x):
        nat.check(nat.lib.flb_layer_norm_fwd(x.data_ptr(), ldx, nat.ptr(w), nat.ptr(b), wdt, y.data_ptr(), nat.ptr(mean),
                                             nat.ptr(rstd), nat.ptr(codes), nat.ptr(exps), G, R, D, dt, eps,
                                             nat.stream_of(x)), "flb_layer_norm_fwd")
    return y, (mean, rstd, codes, exps)


def _backward(x, mean, rstd, codes, exps, weight, bias, dy, dtype):
    """dx, dweight, dbias. x and mean, or codes and exps."""
    dy = dy.to(dtype).contiguous()
    D = dy.shape[-1]
    dt = dtype_of(dy, "dy")
    like = weight if weight is not None else bias
    wdt = dt if like is None else dtype_of(like, "weight")
    G = like.shape[0] if like is not None and like.ndim == 2 else 1
    rows = dy.numel() // D
    R = rows // G if G else 0
    ldx = D
    if x is not None:
        x, ldx = as_rows(x)
    w = None if weight is None else weight.contiguous()
    dx = torch.empty_like(dy)
    dw = db = ws = None
    need = 0
    with on_device_of(dy):
        if like is not None:
            dw = torch.empty(like.shape, dtype=like.dtype, device=dy.device)
            db = torch.empty_like(dw)
            need = nat.lib.flb_layer_norm_bwd_workspace_bytes(G, R, D, dt)
            ws = nat.workspace(need, dy.device)
        nat.check(nat.lib.flb_layer_norm_bwd(nat.ptr(x), ldx, nat.ptr(codes), nat.ptr(exps), nat.ptr(mean), rstd.data_ptr(),
                                             nat.ptr(w), wdt, dy.data_ptr(), dx.data_ptr(), nat.ptr(dw), nat.ptr(db), G, R,
                                             D, dt, nat.ptr(ws), need, nat.stream_of(dy)), "flb_layer_norm_bwd")
    return dx, dw if weight is not None else None, db if bias is not None else None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep8):
        y, kept = _forward(x, weight, bias, eps, keep8, True)
        ctx.dtype = x.dtype
        ctx.save_for_backward(None if keep8 else x, *kept, weight, bias)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return *_backward(*ctx.saved_tensors, dy, ctx.dtype), None, None


class _LayerNormFunc(torch.autograd.Function):
    """The same under torch.func transforms: what the backward reads are outputs of the forward."""

    @staticmethod
    def forward(x, weight, bias, eps, keep8):
        y, (mean, rstd, codes, exps) = _forward(x, weight, bias, eps, keep8, True)
        return (y, rstd, codes, exps) if keep8 else (y, rstd, mean)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, weight, bias, _, ctx.keep8 = inputs
        ctx.dtype = x.dtype
        ctx.mark_non_differentiable(*output[1:])
        ctx.save_for_backward(None if ctx.keep8 else x, weight, bias, *output[1:])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, *_):
        x, weight, bias, rstd, *kept = (plain(t) for t in ctx.saved_tensors)
        mean, codes, exps = (None, *kept) if ctx.keep8 else (kept[0], None, None)
        return *_backward(x, mean, rstd, codes, exps, weight, bias, plain(dy), ctx.dtype), None, None

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
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps), bool(keep8))
    return _forward(x, weight, bias, float(eps), False, False)[0]


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
