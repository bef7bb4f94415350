"""Shared by the row operators' torch.func rules."""
from __future__ import annotations

import torch

transforms_active = torch._C._are_functorch_transforms_active


def no_transforms(what: str) -> None:
    """Refuses torch.func transforms where an operator has no rule for them."""
    if transforms_active():
        raise RuntimeError(f"{what} is not supported under torch.func transforms")


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
