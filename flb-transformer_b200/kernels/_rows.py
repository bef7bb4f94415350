"""Shared by the row operators' torch.func rules."""
from __future__ import annotations

import torch

transforms_active = torch._C._are_functorch_transforms_active


def no_transforms(what: str) -> None:
    """Refuses torch.func transforms where an operator has no rule for them."""
    if transforms_active():
        raise RuntimeError(f"{what} is not supported under torch.func transforms")


NO_VMAP = "vmap over this operator's backward pass is not supported: take the gradient of the vmapped function instead"


def plain(t):
    """The tensor inside torch.func's gradient wrappers. A batched one is refused: its storage holds
    every sample of a vmap that the caller's formula knows nothing of."""
    from torch._C._functorch import get_unwrapped, is_batchedtensor, is_functorch_wrapped_tensor
    while isinstance(t, torch.Tensor) and is_functorch_wrapped_tensor(t):
        if is_batchedtensor(t):
            raise RuntimeError(NO_VMAP)
        t = get_unwrapped(t)
    return t


class once(torch.autograd.Function):
    """A backward pass as a function of its own, for a gradient that is itself differentiated or computed under torch.func
    transforms: each level of torch.func and of autograd sees it, and its own derivative is refused there. once.apply(call,
    *args) returns the tensors that call(*args) does."""

    @staticmethod
    def forward(call, *args):
        return tuple(t for t in call(*args) if t is not None)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("this operator is differentiable once")

    @staticmethod
    def vmap(info, in_dims, *_):
        raise RuntimeError(NO_VMAP)


def backward_of(call, *args):
    """call(*args), an operator's backward pass on plain tensors, from an autograd function's backward method: the
    tensors it returns, without the Nones among them."""
    if torch.is_grad_enabled() or transforms_active():
        return once.apply(call, *args)
    # neither this gradient's graph nor another transform's is wanted
    return tuple(t for t in call(*map(plain, args)) if t is not None)


def to_front(t: torch.Tensor, dim: int | None, size: int) -> torch.Tensor:
    """A vmapped argument with its mapped axis first (expanded where it is not mapped)."""
    return t.unsqueeze(0).expand(size, *t.shape) if dim is None else t.movedim(dim, 0)
