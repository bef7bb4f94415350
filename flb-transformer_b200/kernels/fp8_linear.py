"""Linear maps in 8-bit floating point with a power of two for each block of 128, on B200 (sm_100a).

    quantize_fp8(x) -> Fp8Rows
    fp8_linear(x, weight, bias=None, check_timeout=False) -> x @ weight.T + bias
    Fp8Linear(in, out), Fp8Linear.from_linear(linear)      an nn.Linear that calls it, for training
    .kept() -> Fp8LinearKept                               its weight in 8 bits once and for all, for inference

A block of 128 consecutive elements of a row is held as e4m3 codes (4 significant bits, magnitudes up to 448) in units
of the smallest power of two, from 2^-127 on, in which its largest magnitude is at most 448. An element is off by at
most 1/16 of itself, or where it is below 2^-6 units, 2^-10 units (of float32, one above 1.93 * 2^127 counts as 2^128, an
infinity). A block that holds an infinity or NaN counts as NaN.
Against 8-bit integers with a scale a row (int8_linear) small elements keep their precision beside large ones, and
an outlier costs the others of its block nothing until it is 2^15 times as large.

With a plain weight [N, K] the map is differentiable once in x, weight and bias. Its gradients are products of the same
kind, each operand in blocks along the axis that is summed: dx = dy W with both along the outputs, dW = dy.T x with both
along the tokens; db is the plain sum of dy. x and W are kept for the backward pass in 8 bits. With a weight in Fp8Rows
there are no gradients. Products are in float32: over 1024 of K as the tensor core adds, which cuts, and between
those rounded. The same inputs give the same bits.

The kernels' waits for their own copies and products are bounded (4 s). Where one gave up, the outputs (or gradients) that
it held up are NaN. check_timeout (inference only) also waits for the product and raises a RuntimeError then; without it
the call returns at once.

The kernels are in libflb_b200.so (flb_fp8_rows, flb_fp8_rows2, flb_fp8_linear: tcgen05 kind::mxf8f6f4), called through
flb_ops; CUDA tensors only. torch.func transforms are refused.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

import flb_native  # noqa: F401  (loads libflb_b200.so, or says that it is missing)
import flb_ops
from ._rows import no_transforms

__all__ = ["Fp8Rows", "quantize_fp8", "fp8_linear", "Fp8Linear", "Fp8LinearKept"]


class Fp8Rows(NamedTuple):
    """Rows in 8-bit floating point: codes float8_e4m3fn [..., K], exps uint8 [ceil(rows / 128), ceil(K / 512), 32, 4, 4] (of
    row r and block b at [r // 128, b // 4, r % 32, r // 32 % 4, b % 4], with 2 ** (byte - 127) as the unit; zeros in
    other places), and the type they had. Codes whose rows start on 16 bytes, as quantize_fp8 lays them out, are read in
    place; others are copied by every call that reads them."""
    codes: torch.Tensor
    exps: torch.Tensor
    dtype: torch.dtype = torch.bfloat16

    def units(self) -> torch.Tensor:
        """Each block's unit, float32 [..., ceil(K / 128)]; NaN for a block that held an infinity or NaN."""
        shape = self.codes.shape
        rows, blocks = self.codes[..., 0].numel(), -(-shape[-1] // 128)
        e = self.exps.permute(0, 3, 2, 1, 4).reshape(self.exps.shape[0] * 128, self.exps.shape[1] * 4)[:rows, :blocks]
        e = torch.where(e == 255, torch.nan, torch.exp2(e.double() - 127)).float()
        return e.reshape(*shape[:-1], blocks)

    def dequantize(self) -> torch.Tensor:
        """The values that the rows stand for, in float32."""
        K = self.codes.shape[-1]
        return self.codes.float() * self.units().repeat_interleave(128, -1)[..., :K]


def quantize_fp8(x: torch.Tensor) -> Fp8Rows:
    """x [..., K] (float32, float16 or bfloat16) with each row of its last axis in 8-bit floating point: a token's features, or
    (x a weight [out, in]) an output channel's."""
    no_transforms("quantize_fp8")
    return Fp8Rows(*flb_ops.quantize_fp8(x), x.dtype)


def fp8_linear(x: torch.Tensor | Fp8Rows, weight: torch.Tensor | Fp8Rows, bias: torch.Tensor | None = None,
               check_timeout: bool = False) -> torch.Tensor:
    """x [..., K] times weight [N, K], plus bias [N]: [..., N] in x's type, also under autocast. weight and bias: float32, float16 or bfloat16; the
    weight as a plain tensor (differentiable), or in Fp8Rows (inference; then x may be so too). See the module's text."""
    no_transforms("fp8_linear")
    if not isinstance(weight, Fp8Rows):
        if isinstance(x, Fp8Rows) or check_timeout:
            raise ValueError("x in 8 bits and check_timeout need a weight in 8 bits (quantize_fp8)")
        return flb_ops.fp8_linear(x, weight, bias)
    if isinstance(x, Fp8Rows):
        return flb_ops.fp8_linear_kept(None, x.codes, x.exps, weight.codes, weight.exps, bias, x.dtype, check_timeout)
    return flb_ops.fp8_linear_kept(x, None, None, weight.codes, weight.exps, bias, None, check_timeout)


class Fp8Linear(nn.Linear):
    """nn.Linear with the same parameters, whose product and its gradients are fp8_linear's: the weight goes into 8 bits in each
    forward pass, as a training step's must."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp8_linear(x, self.weight, self.bias)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Fp8Linear":
        """A map with the same parameters (not copies)."""
        out = cls(linear.in_features, linear.out_features, linear.bias is not None, device="meta")
        out.weight, out.bias = linear.weight, linear.bias
        return out

    @torch.no_grad()
    def kept(self, check_timeout: bool = False) -> "Fp8LinearKept":
        """The map for inference, with its weight as it is now."""
        return Fp8LinearKept(quantize_fp8(self.weight), None if self.bias is None else self.bias.detach().clone(), check_timeout)


class Fp8LinearKept(nn.Module):
    """A linear map whose weight is kept in 8-bit floating point (buffers `codes` and `exps`, which keep their types when the module is
    cast). For inference: its output has no gradient. check_timeout as in fp8_linear."""

    def __init__(self, weight: Fp8Rows, bias: torch.Tensor | None = None, check_timeout: bool = False):
        super().__init__()
        self.check_timeout = check_timeout
        self.out_features, self.in_features = weight.codes.shape
        self.register_buffer("codes", weight.codes)
        self.register_buffer("exps", weight.exps)
        self.register_buffer("bias", bias)

    def _apply(self, fn, recurse=True):
        # a cast of the model is not for the codes: they follow to its device alone
        kept = {"codes": self.codes, "exps": self.exps}
        super()._apply(fn, recurse)
        for name, t in kept.items():
            moved = getattr(self, name)
            if moved.dtype != t.dtype:
                setattr(self, name, t.to(moved.device))
        return self

    @torch.no_grad()
    def forward(self, x: torch.Tensor | Fp8Rows) -> torch.Tensor:
        return fp8_linear(x, Fp8Rows(self.codes, self.exps), self.bias, self.check_timeout)
