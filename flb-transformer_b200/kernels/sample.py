"""The choice of a token from logits on B200 (sm_100a).

    sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> tokens

With w_i = exp((l_i - max l) / temperature) along a row of logits:
  top_k   keeps the top_k tokens of the largest logits, of equal ones those of lower index (0: all),
  top_p   of these the shortest run from the largest on whose w sum to at least top_p of theirs (always the
          first; 1: all),
  min_p   of these the ones with w_i >= min_p: of at least min_p of the largest one's probability,
and the token is the first, in the vocabulary's order, at which the sum of kept w passes u of the whole. u, one
uniform number in [0, 1) a row, is all the randomness there is: the same u gives the same token. A temperature of 0
gives the largest logit, of equal ones the lowest index. A row whose logits are all -inf (all masked), or with a NaN
among them, gives -1; logits of +inf share all of the probability.

Weights are float64 and summed as 64-bit integers in units of 2^-47 (at 32000 tokens; 2^-44 at 262144), each within
4e-14 of itself and half a unit of the definition's: over normal logits at most 7 draws in 10^9 gave another
token than the definition, 7 in 10^6 at 262144. Vocabularies of up to 262144. The kernel is in libflb_b200.so (flb_sample),
called through flb_ops; CUDA tensors only.
"""
from __future__ import annotations

from operator import index

import torch

import flb_native  # noqa: F401  (loads libflb_b200.so, or says that it is missing)
import flb_ops
from ._rows import no_transforms

__all__ = ["sample"]


def _rows_or_all(value, whole=float):
    return (value, whole(0)) if isinstance(value, torch.Tensor) else (None, whole(value))


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: float | torch.Tensor = 1.0, top_k: int | torch.Tensor = 0,
           top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0) -> torch.Tensor:
    """logits [..., V] (float32, float16 or bfloat16) and u [...] (float32 or float64) -> int64 [...]. Each setting is a
    number for all rows, or a tensor [...] with one a row (float32; top_k int64). See the module's text."""
    no_transforms("sample")
    return flb_ops.sample(logits, u, *_rows_or_all(temperature), *_rows_or_all(top_k, index), *_rows_or_all(top_p), *_rows_or_all(min_p))
