"""Activations kept in 8 bits between forward and backward, and the sigmoid gate that keeps its inputs so.

    pack8(x) -> Packed8, unpack8(p) -> tensor
    sigmoid_gate(x, z, keep8=False) -> x * sigmoid(z)

The kept form holds blocks of 128 consecutive elements of the last axis as integers of at most 127 in
magnitude times a power of two, the smallest for which the block's largest magnitude still rounds to at
most 127: an element is off by at most 1/127 of its block's largest magnitude (half a unit of between
1/127.5 and 1/63.5 of it). That holds for largest magnitudes from 63.5 * 2^-126 to 63.5 * 2^122 (7.5e-37 to
3.38e38). Below, the unit stays 2^-126: an element is off by at most 2^-127, and a block of less than that
comes back as zeros. Above, where float32 does not hold a code of 64, it is 63: off by at most 1/63 of the
largest magnitude. A block that holds an infinity or NaN comes back as NaN. It takes 1 + 1/128 bytes an
element (the rows of codes padded to 16 bytes).

The kernels are in libflb_b200.so (flb_pack8, flb_unpack8, flb_gate_fwd, flb_gate_bwd), called through
flb_ops; CUDA tensors only.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

import flb_native  # noqa: F401  (loads libflb_b200.so, or says that it is missing)
import flb_ops
from ._rows import backward_of, no_transforms, to_front, transforms_active

__all__ = ["Packed8", "pack8", "unpack8", "sigmoid_gate"]


class Packed8(NamedTuple):
    """A tensor's kept form: codes int8 [rows, pitch], exps uint8 [rows, blocks], and what it was."""
    codes: torch.Tensor
    exps: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype


def pack8(x: torch.Tensor) -> Packed8:
    """The kept form of x (float32, float16 or bfloat16, any shape with at least one axis). Not
    differentiable: it is what an operator's forward keeps for its backward."""
    no_transforms("pack8")
    return Packed8(*flb_ops.pack8(x.detach()), x.shape, x.dtype)


def unpack8(p: Packed8, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The tensor that p stands for, in its own type or `dtype` (float16 saturates)."""
    no_transforms("unpack8")
    return flb_ops.unpack8(p.codes, p.exps, list(p.shape), dtype or p.dtype)


class _GateFunc(torch.autograd.Function):
    """The gate under torch.func transforms: what the backward reads are outputs of the forward."""

    @staticmethod
    def forward(x, z, keep8):
        # with keep8 an empty tensor last, which tells the levels of torch.func that the kept forms (integers) depend on x and z
        return (*flb_ops.gate_forward(x, z, keep8), *([x.new_empty(0)] if keep8 else []))

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, z, keep8 = inputs
        ctx.mark_non_differentiable(*output[1:-1])
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*(output[1:] if keep8 else (x, z)))

    @staticmethod
    def backward(ctx, dy, *_):
        return *backward_of(lambda dy, *kept: flb_ops.gate_backward(list(kept[:4]), dy), dy, *ctx.saved_tensors), None

    @staticmethod
    def vmap(info, in_dims, x, z, keep8):
        x, z = (to_front(t, d, info.batch_size) for t, d in zip((x, z), in_dims))
        out = _GateFunc.apply(x, z, keep8)
        # the kept forms' rows are not split by sample: they only travel to the backward
        return out, (0, *(None,) * (len(out) - 1))


def sigmoid_gate(x: torch.Tensor, z: torch.Tensor, keep8: bool = False) -> torch.Tensor:
    """x * sigmoid(z), x and z of one shape and type. With keep8 the backward reads x and z from 8 bits
    (the output is the same). Differentiable once; torch.vmap is supported."""
    if transforms_active():
        return _GateFunc.apply(x, z, bool(keep8))[0]
    return flb_ops.sigmoid_gate(x, z, keep8)
