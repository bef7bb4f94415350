"""Activations kept in 8 bits between forward and backward, and the sigmoid gate that keeps its inputs so.

    pack8(x) -> Packed8, unpack8(p) -> tensor
    sigmoid_gate(x, z, keep8=False) -> x * sigmoid(z)

The kept form holds blocks of 128 consecutive elements of the last axis as integers of at most 127 in
magnitude times a power of two, the smallest for which the block's largest magnitude still rounds to at
most 127: an element is off by at most 1/127 of its block's largest magnitude (half a unit of between
1/127.5 and 1/63.5 of it). A block that holds an infinity or NaN comes back as NaN. It takes
1 + 1/128 bytes an element (the rows of codes padded to 16 bytes).

The kernels are in libflb_b200.so (flb_pack8, flb_unpack8, flb_gate_fwd, flb_gate_bwd); CUDA tensors only.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

import flb_native as nat
from ._rows import dtype_of, on_device_of, plain, same_device, to_front, transforms_active

__all__ = ["Packed8", "pack8", "unpack8", "sigmoid_gate"]


class Packed8(NamedTuple):
    """A tensor's kept form: codes int8 [rows, pitch], exps uint8 [rows, blocks], and what it was."""
    codes: torch.Tensor
    exps: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype


def kept_buffers(rows: int, D: int, device):
    """Empty codes and exps for `rows` rows of D elements."""
    return (torch.empty((rows, (D + 15) // 16 * 16), dtype=torch.int8, device=device),
            torch.empty((rows, (D + 127) // 128), dtype=torch.uint8, device=device))


def _rows_of(shape):
    if not shape:
        raise ValueError("a tensor with at least one axis is needed")
    D = shape[-1]
    rows = 1
    for n in shape[:-1]:
        rows *= n
    return rows, D


def pack8(x: torch.Tensor) -> Packed8:
    """The kept form of x (float32, float16 or bfloat16, any shape with at least one axis). Not
    differentiable: it is what an operator's forward keeps for its backward."""
    dt = dtype_of(x, "x")
    same_device(x)
    rows, D = _rows_of(x.shape)
    x_ = x.detach().contiguous()
    codes, exps = kept_buffers(rows, D, x.device)
    if rows and D:
        with on_device_of(x):
            nat.check(nat.lib.flb_pack8(x_.data_ptr(), codes.data_ptr(), exps.data_ptr(), rows, D, dt,
                                        nat.stream_of(x)), "flb_pack8")
    return Packed8(codes, exps, x.shape, x.dtype)


def unpack8(p: Packed8, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The tensor that p stands for, in its own type or `dtype`."""
    shape = torch.Size(p.shape)
    rows, D = _rows_of(shape)
    if (p.codes.dtype != torch.int8 or p.exps.dtype != torch.uint8
            or tuple(p.codes.shape) != (rows, (D + 15) // 16 * 16) or tuple(p.exps.shape) != (rows, (D + 127) // 128)
            or not p.codes.is_contiguous() or not p.exps.is_contiguous()):
        raise ValueError("codes and exps are not a kept form of shape " + str(tuple(shape)))
    same_device(p.codes, p.exps)
    out = torch.empty(shape, dtype=dtype or p.dtype, device=p.codes.device)
    dt = dtype_of(out, "the type")
    if rows and D:
        with on_device_of(out):
            nat.check(nat.lib.flb_unpack8(p.codes.data_ptr(), p.exps.data_ptr(), out.data_ptr(), rows, D, dt,
                                          nat.stream_of(out)), "flb_unpack8")
    return out


def _gate_forward(x, z, keep8):
    dt = dtype_of(x, "x")
    same_device(x, z)
    if x.shape != z.shape:
        raise ValueError(f"x and z differ in shape: {tuple(x.shape)} {tuple(z.shape)}")
    if z.dtype != x.dtype:
        raise TypeError(f"x and z differ in type: {x.dtype} {z.dtype}")
    rows, D = _rows_of(x.shape)
    x, z = x.contiguous(), z.contiguous()
    y = torch.empty_like(x)
    kept = (*kept_buffers(rows, D, x.device), *kept_buffers(rows, D, x.device)) if keep8 else (None,) * 4
    if rows and D:
        with on_device_of(x):
            nat.check(nat.lib.flb_gate_fwd(x.data_ptr(), z.data_ptr(), y.data_ptr(), *map(nat.ptr, kept), rows, D,
                                           dt, nat.stream_of(x)), "flb_gate_fwd")
    return y, kept


def _gate_backward(x, z, kept, dy, dtype):
    """x, z: the inputs, or None with `kept` their kept forms."""
    dy = dy.to(dtype).contiguous()
    rows, D = _rows_of(dy.shape)
    if x is not None:
        x, z = x.contiguous(), z.contiguous()
    dx, dz = torch.empty_like(dy), torch.empty_like(dy)
    if rows and D:
        with on_device_of(dy):
            nat.check(nat.lib.flb_gate_bwd(nat.ptr(x), nat.ptr(z), *map(nat.ptr, kept), dy.data_ptr(), dx.data_ptr(),
                                           dz.data_ptr(), rows, D, dtype_of(dy, "dy"), nat.stream_of(dy)),
                      "flb_gate_bwd")
    return dx, dz


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, keep8):
        y, kept = _gate_forward(x, z, keep8)
        ctx.keep8, ctx.dtype = keep8, x.dtype
        ctx.save_for_backward(*(kept if keep8 else (x, z)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        t = ctx.saved_tensors
        if ctx.keep8:
            return *_gate_backward(None, None, t, dy, ctx.dtype), None
        return *_gate_backward(t[0], t[1], (None,) * 4, dy, ctx.dtype), None


class _GateFunc(torch.autograd.Function):
    """The same under torch.func transforms: what the backward reads are outputs of the forward."""

    @staticmethod
    def forward(x, z, keep8):
        y, kept = _gate_forward(x, z, keep8)
        return (y, *kept) if keep8 else y

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, z, ctx.keep8 = inputs
        ctx.dtype = x.dtype
        if ctx.keep8:
            ctx.mark_non_differentiable(*output[1:])
            ctx.save_for_backward(*output[1:])
        else:
            ctx.save_for_backward(x, z)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, *_):
        t = [plain(s) for s in ctx.saved_tensors]
        dy = plain(dy)
        if ctx.keep8:
            return *_gate_backward(None, None, t, dy, ctx.dtype), None
        return *_gate_backward(t[0], t[1], (None,) * 4, dy, ctx.dtype), None

    @staticmethod
    def vmap(info, in_dims, x, z, keep8):
        x, z = (to_front(t, d, info.batch_size) for t, d in zip((x, z), in_dims))
        out = _GateFunc.apply(x, z, keep8)
        # the kept forms' rows are not split by sample: they only travel to the backward
        return out, ((0, None, None, None, None) if keep8 else 0)


def sigmoid_gate(x: torch.Tensor, z: torch.Tensor, keep8: bool = False) -> torch.Tensor:
    """x * sigmoid(z), x and z of one shape and type. With keep8 the backward reads x and z from 8 bits
    (the output is the same). Differentiable once; torch.vmap is supported."""
    if transforms_active():
        out = _GateFunc.apply(x, z, bool(keep8))
        return out[0] if keep8 else out
    if torch.is_grad_enabled() and (x.requires_grad or z.requires_grad):
        return _Gate.apply(x, z, bool(keep8))
    return _gate_forward(x, z, False)[0]
