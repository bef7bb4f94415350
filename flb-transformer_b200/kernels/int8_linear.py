"""Linear maps in 8-bit integers with a scale for each token and each output channel, on B200 (sm_100a).

    quantize_int8(x) -> Int8Rows
    int8_linear(x, weight, bias=None, check_timeout=False) -> x @ weight.T + bias
    Int8Linear.from_linear(linear)                       a module with its weight so quantised

A row v is codes round(v * 127 / max|v|) and the scale max|v| / 127; int8_linear makes its input's rows so on the
way (or takes them as Int8Rows, as layer_norm_int8 returns them), adds products of codes in 32-bit
integers, without rounding, and multiplies by the two scales. A row that holds an infinity or NaN gives
NaN in all its outputs; one whose largest magnitude is below 2^-118 counts as zeros. Rows of up to 32768
elements. No gradients: inference only.

The kernels' waits for their own copies and products are bounded (4 s). check_timeout waits for the product and raises a
RuntimeError if one of them gave up, where the output is wrong; without it the call returns at once and nothing is said.

The kernels are in libflb_b200.so (flb_int8_rows, flb_int8_linear: tcgen05 kind::i8), called through
flb_ops; CUDA tensors only.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

import flb_native  # noqa: F401  (loads libflb_b200.so, or says that it is missing)
import flb_ops
from ._rows import no_transforms

__all__ = ["Int8Rows", "quantize_int8", "int8_linear", "Int8Linear"]


class Int8Rows(NamedTuple):
    """Rows in 8-bit integers: codes int8 [..., K], scale float32 [...], and the type they had. Codes whose
    rows start on 16 bytes, as quantize_int8 lays them out, are read in place; others are copied by every
    call that reads them."""
    codes: torch.Tensor
    scale: torch.Tensor
    dtype: torch.dtype = torch.bfloat16

    def dequantize(self) -> torch.Tensor:
        """The values that the rows stand for, in float32."""
        return self.codes.float() * self.scale[..., None]


def quantize_int8(x: torch.Tensor) -> Int8Rows:
    """x [..., K] (float32, float16 or bfloat16) with each row of its last axis in 8-bit integers: a token's
    features, or (x a weight [out, in]) an output channel's."""
    no_transforms("quantize_int8")
    return Int8Rows(*flb_ops.quantize_int8(x), x.dtype)


def int8_linear(x: torch.Tensor | Int8Rows, weight: Int8Rows, bias: torch.Tensor | None = None,
                check_timeout: bool = False) -> torch.Tensor:
    """x [..., K] times weight [N, K] (an Int8Rows), plus bias [N] (float32 or x's type): [..., N] in x's type.
    check_timeout: see the module's text; not while a CUDA graph is captured."""
    no_transforms("int8_linear")
    if isinstance(x, Int8Rows):
        return flb_ops.int8_linear(None, x.codes, x.scale, weight.codes, weight.scale, bias, x.dtype, check_timeout)
    return flb_ops.int8_linear(x, None, None, weight.codes, weight.scale, bias, None, check_timeout)


class Int8Linear(nn.Module):
    """A linear map whose weight is kept in 8-bit integers (buffers `codes` and `scale`, which keep their types when the module
    is cast). For inference: its output has no gradient. check_timeout as in int8_linear."""

    def __init__(self, weight: Int8Rows, bias: torch.Tensor | None = None, check_timeout: bool = False):
        super().__init__()
        self.check_timeout = check_timeout
        self.out_features, self.in_features = weight.codes.shape
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scale", weight.scale)
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, linear: nn.Linear, check_timeout: bool = False) -> "Int8Linear":
        """The map of an nn.Linear on a CUDA device, with its weight as it is now."""
        with torch.no_grad():
            bias = None if linear.bias is None else linear.bias.detach().clone()
            return cls(quantize_int8(linear.weight), bias, check_timeout)

    def _apply(self, fn, recurse=True):
        # a cast of the model is not for the codes and scales: they follow to its device alone
        kept = {"codes": self.codes, "scale": self.scale}
        super()._apply(fn, recurse)
        for name, t in kept.items():
            moved = getattr(self, name)
            if moved.dtype != t.dtype:
                setattr(self, name, t.to(moved.device))
        return self

    @torch.no_grad()
    def forward(self, x: torch.Tensor | Int8Rows) -> torch.Tensor:
        bias = self.bias
        if bias is not None and bias.dtype not in (torch.float32, x.dtype):
            bias = bias.float()
        return int8_linear(x, Int8Rows(self.codes, self.scale), bias, self.check_timeout)
