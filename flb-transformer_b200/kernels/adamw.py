"""AdamW on B200 (sm_100a): one kernel for all of a model's tensors, moments in 32 or in 8 bits.

    opt = AdamW(params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0)

    m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr weight_decay) - lr (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps)

in float32, p (float32, float16 or bfloat16) rounded once. A torch.optim.Optimizer: groups, schedulers and state dicts
as there, and the names of its state ("step", "exp_avg", "exp_avg_sq").

state_bits=8 holds the moments in 8-bit floating point, blocks of 128 elements each with a byte for the exponent of its
largest magnitude ("exp_avg_exps", "exp_avg_sq_exps"): m with a sign, 3 bits of mantissa and the 16 binades
around and under the block's largest, v with 3 bits of mantissa and 32 binades. 2 bytes an element instead of 8. They are
rounded up or down at random (a mix of the element's index, the step and `seed`: the same every time, and the same for every
tensor), so that a moment that changes by less than its unit a step still follows its mean. One element's v
then stands off its exact value by about 20% (root of the mean square; 26% with gradients of which nine in ten are zero; between
0.3 and 3 times it over 16384 elements, beta2 = 0.999), so its update by about half of that; the mean is right to 0.2%. Below the smallest code m becomes zero, and v the
smallest code. A block with an infinity or NaN becomes NaN as a whole. Blocks and codes go by the parameter's memory, whose
strides are in the state ("strides") of one that is not contiguous: a state goes into, and on with, a parameter that is laid out
the same, and into another one is refused. (Moments in 32 bits are loaded by element.)

Steps are counted on the device, each tensor's own (its "step", an int64), so that a captured step counts on in every replay;
lr may be a float32 tensor on the device, which a schedule then writes between replays. The first step of a tensor makes its
state, and is not for a capture; with state that was loaded or copied a capture may be an optimizer's first step. Steps of one optimizer must not overlap on the GPU. The kernels are in libflb_b200.so
(flb_adamw, flb_adamw_moments), called through flb_ops; CUDA tensors only.
"""
from __future__ import annotations

import torch

import flb_native  # noqa: F401  (loads libflb_b200.so, or says that it is missing)
import flb_ops

__all__ = ["AdamW"]


class AdamW(torch.optim.Optimizer):
    """See the module's text."""

    def __init__(self, params, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, seed: int = 0):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            self._check(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group):
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or (lr.is_cuda and lr.dtype != torch.float32):
                raise ValueError("lr must be a number, or a tensor of one float32")
        elif not lr >= 0:
            raise ValueError(f"lr must be at least 0, not {lr}")
        if not (0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError(f"betas must be at least 0 and below 1, not {group['betas']}")
        if not (group["eps"] >= 0 and group["weight_decay"] >= 0):
            raise ValueError("eps and weight_decay must be at least 0")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {group['state_bits']}")
        for name in ("maximize", "amsgrad"):
            if group.get(name):
                raise ValueError(f"AdamW has no {name}")
        if group["weight_decay"] > 0 and not group.get("decoupled_weight_decay", True):
            raise ValueError("AdamW's weight_decay is decoupled from the moments (decoupled_weight_decay=False)")
        if len(set(map(id, group["params"]))) != len(group["params"]):
            raise ValueError("a parameter is in the group twice")
        for p in group["params"]:
            if p.dtype not in (torch.float32, torch.float16, torch.bfloat16):
                raise TypeError(f"parameters must be float32, float16 or bfloat16, not {p.dtype}")

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("state_bits", 32)
            group.setdefault("seed", 0)
        # State that was loaded or copied may take its first step in a capture, which must not make the kernel's word on its device.
        counters = self.__dict__.setdefault("_counters", {})
        for p, s in self.__dict__.get("state", {}).items():
            if s and isinstance(p, torch.Tensor) and p.is_cuda and p.device.index not in counters and not torch.cuda.is_current_stream_capturing():
                counters[p.device.index] = torch.zeros(1, dtype=torch.int32, device=p.device)

    def _new_state(self, p, bits):
        state = {"step": torch.zeros((), dtype=torch.int64, device=p.device)}
        blocks = -(-p.numel() // 128)
        if bits == 8 and not p.is_contiguous():
            state["strides"] = p.stride()
        for name in ("exp_avg", "exp_avg_sq"):
            if bits == 8:
                state[name] = torch.zeros(blocks, 128, dtype=torch.uint8, device=p.device)
                state[name + "_exps"] = torch.zeros(blocks, dtype=torch.uint8, device=p.device)
            else:
                state[name] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        return state

    @staticmethod
    def _check_order(s, p):
        """Refuses 8-bit state of a parameter that was laid out otherwise. (Axes of one element have no place in memory.)"""
        strides = s.get("strides")
        same = p.is_contiguous() if strides is None else len(strides) == p.dim() and all(
            n == 1 or a == b for n, a, b in zip(p.shape, strides, p.stride()))
        if not same:
            raise ValueError(f"8-bit moments are not laid out as their parameter, of shape {tuple(p.shape)} and strides {p.stride()}")

    @torch.no_grad()
    def step(self, closure=None):
        """One step of every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        counters = self.__dict__.setdefault("_counters", {})
        for group in self.param_groups:
            lr = group["lr"]
            on_device = isinstance(lr, torch.Tensor) and lr.is_cuda
            args = (group["params"], self.state, group["state_bits"], 0.0 if on_device else float(lr), lr.detach() if on_device else None,
                    *group["betas"], group["eps"], group["weight_decay"], group["seed"] & 0xffffffff, counters)
            new = flb_ops.adamw(*args)
            if new:
                for p in new:
                    if not p.is_cuda:
                        raise RuntimeError(f"AdamW runs on CUDA tensors only (sm_100a kernels; no CPU path); got a parameter on {p.device}")
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamW: the first step of a parameter makes its state: take one before the capture")
                try:
                    for p in new:
                        self.state[p].update(self._new_state(p, group["state_bits"]))
                    flb_ops.adamw(*args)
                except Exception:
                    for p in new:  # a step that was refused was not the first one
                        self.state.pop(p, None)
                    raise
        return loss

    @torch.no_grad()
    def moments(self, out=None) -> list:
        """(m, v) of every parameter that has taken a step, in the groups' order, as float32 tensors of its shape. Of 32 bits they are the
        state's own; of 8 bits new ones, or those of `out`, a list of such pairs of contiguous tensors, written."""
        found = []
        if out is not None and len(out) != sum(1 for group in self.param_groups for p in group["params"] if self.state.get(p)):
            raise ValueError("`out` does not have a pair for each parameter that has taken a step")
        for group in self.param_groups:
            if group["state_bits"] == 8:
                found += flb_ops.adamw_moments(group["params"], self.state, out, len(found))
                continue
            for p in group["params"]:
                if not self.state.get(p):
                    continue
                pair = (self.state[p]["exp_avg"], self.state[p]["exp_avg_sq"])
                if out is not None:
                    for to, x in zip(out[len(found)], pair):
                        to.copy_(x)
                    pair = tuple(out[len(found)])
                found.append(pair)
        return found

    @staticmethod
    def _check_state(s, p, bits):
        """Refuses state that is not a parameter's of p's shape: copied in, it could be repeated to fill it."""
        if ("exp_avg_exps" in s) != (bits == 8):
            raise ValueError("the state's moments are not of the bits that its group says")
        blocks = -(-p.numel() // 128)
        want = {"step": None}
        for name in ("exp_avg", "exp_avg_sq"):
            want.update({name: (blocks, 128), name + "_exps": (blocks,)} if bits == 8 else {name: tuple(p.shape)})
        for name, shape in want.items():
            if name not in s:
                raise ValueError(f"the state has no {name}")
            t = torch.as_tensor(s[name])
            if t.numel() != 1 if shape is None else tuple(t.shape) != shape or (bits == 8 and t.dtype != torch.uint8):
                raise ValueError(f"the state's {name}, of shape {tuple(t.shape)} and {t.dtype}, is not that of a parameter of shape {tuple(p.shape)}")
        if bits == 8:
            AdamW._check_order(s, p)

    def _check_saved(self, state_dict):
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            saved = {"state_bits": 32, "seed": 0, **saved}
            self._check({**saved, "params": group["params"]})
            for p, key in zip(group["params"], saved["params"]):
                if state_dict["state"].get(key):
                    self._check_state(state_dict["state"][key], p, saved["state_bits"])

    def _take_state(self, state_dict):
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], saved["params"]):
                if not state_dict["state"].get(key):
                    continue
                s, mine = state_dict["state"][key], self._new_state(p, group["state_bits"])
                for name, t in mine.items():
                    if isinstance(t, torch.Tensor):
                        t.copy_(torch.as_tensor(s[name]).reshape(t.shape))
                self.state[p] = mine

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, but the state keeps its types. Moments in 32 bits may come from torch.optim.AdamW. What is refused leaves the
        optimizer as it was."""
        final = []

        # the last of the hooks before the load, which see and may replace the dict, and the first of those after it
        def check(_, saved):
            self._check_saved(saved)
            final.append(saved)

        hooks = [self.register_load_state_dict_pre_hook(check), self.register_load_state_dict_post_hook(lambda _: self._take_state(final[0]), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
