"""Shared by the row operators: rows of a tensor as the kernels take them, devices, functorch."""
from __future__ import annotations

import torch

import flb_native as nat

_FLOATS = {torch.float32: nat.F32, torch.float16: nat.F16, torch.bfloat16: nat.BF16}
transforms_active = torch._C._are_functorch_transforms_active


def dtype_of(t: torch.Tensor, what: str) -> int:
    code = _FLOATS.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def as_rows(x: torch.Tensor):
    """(x or a contiguous copy of it, row pitch in elements) with x's leading axes as one axis of rows."""
    D = x.shape[-1]
    if x.is_contiguous():
        return x, D
    if x.stride(-1) == 1 and x.numel() > 0:
        pitch, span = None, None
        for n, s in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
            if n == 1:
                continue
            if pitch is None:
                pitch, span = s, s * n
            elif s == span:
                span *= n
            else:
                return x.contiguous(), D
        return x, D if pitch is None else pitch
    return x.contiguous(), D


def same_device(x: torch.Tensor, *others: torch.Tensor | None) -> None:
    if not x.is_cuda:
        nat.require_cuda(x)
    for t in others:
        if t is not None and t.device != x.device:
            nat.require_cuda(t)
            raise ValueError(f"tensors on different devices: {x.device} and {t.device}")


class on_device_of:
    """Makes x's device the current one, which the library launches on, where it is not already."""

    def __init__(self, x: torch.Tensor):
        self.index = x.device.index
        self.before = -1

    def __enter__(self):
        if self.index != torch._C._cuda_getDevice():
            self.before = torch.cuda._exchange_device(self.index)

    def __exit__(self, *exc):
        if self.before >= 0:
            torch.cuda._maybe_exchange_device(self.before)
        return False


def plain(t):
    """The tensor inside torch.func's gradient wrappers. A batched one is refused: its storage holds
    every sample of a vmap that the caller's formula knows nothing of."""
    from torch._C._functorch import get_unwrapped, is_batchedtensor, is_functorch_wrapped_tensor
    while isinstance(t, torch.Tensor) and is_functorch_wrapped_tensor(t):
        if is_batchedtensor(t):
            raise RuntimeError("vmap over this operator's backward pass is not supported: "
                               "take the gradient of the vmapped function instead")
        t = get_unwrapped(t)
    return t


def to_front(t: torch.Tensor, dim: int | None, size: int) -> torch.Tensor:
    """A vmapped argument with its mapped axis first (expanded where it is not mapped)."""
    return t.unsqueeze(0).expand(size, *t.shape) if dim is None else t.movedim(dim, 0)
