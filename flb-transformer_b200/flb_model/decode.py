"""Decoding for FLBTransformer (the reference has no decode API): greedy, and by sampling.

The model's grid has a fixed width seq_len and its carried contexts reach no cell (the
engine's routing never reads the boundary dock), so a step re-runs the whole grid over the
last seq_len tokens (a sliding window) and appends a token chosen from the last position's logits.
With `graphed=True` the engine's forward tick loop is captured once as a CUDA graph and every
step is one graph replay. With `head` (kernels.Int8Linear.from_linear(model.head), or a
kernels.Fp8Linear's kept()) a step's logits come from it, and for the last position alone.
"""
from __future__ import annotations

import torch

from kernels import sample


def _decode(model, prompt, steps, choose, graphed, engine, head):
    """choose(logits [batch, vocab], step) -> tokens [batch]."""
    from wavefront.wavefront_graph import GraphedWavefrontEngine
    if prompt.dim() != 2 or prompt.shape[1] != model.config.grid_shape[1]:
        raise ValueError(f"prompt must be [batch, {model.config.grid_shape[1]}]")
    window = prompt.clone()
    if engine is None and graphed and steps > 0:
        x = model.emb_dropout(model.embedding(window))
        engine = GraphedWavefrontEngine(model.engine, x, backward=False)
    out = torch.empty(prompt.shape[0], steps, dtype=prompt.dtype, device=prompt.device)
    for s in range(steps):
        if head is None:
            logits, _, _ = model(window, engine=engine)
            nxt = choose(logits[:, -1], s)
        else:
            logits, _, _ = model(window, engine=engine, head=lambda top: head(top[:, -1]))
            nxt = choose(logits, s)
        out[:, s] = nxt
        # (a row without a token, -1, goes on with token 0: the embedding has no row for it)
        window = torch.cat([window[:, 1:], nxt.clamp(min=0)[:, None]], dim=1)
    return out


@torch.no_grad()
def greedy_decode(model, prompt: torch.Tensor, steps: int, graphed: bool = True, engine=None,
                  head=None):
    """prompt [batch, seq_len] int64 token ids -> [batch, steps] generated ids. `engine` may
    pass in a GraphedWavefrontEngine captured earlier (for repeated decodes), `head` a map from
    the hidden states to logits that takes the place of model.head."""
    return _decode(model, prompt, steps, lambda logits, s: logits.argmax(-1), graphed, engine, head)


@torch.no_grad()
def sample_decode(model, prompt: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0, graphed: bool = True, engine=None, head=None):
    """prompt [batch, seq_len] int64 token ids and u [steps, batch], a uniform number in [0, 1) for
    each token -> [batch, steps] ids, chosen by kernels.sample with its settings (numbers, or tensors of
    one a sequence). A step whose logits hold a NaN, or nothing above -inf, gives -1 for its sequence, which
    goes on with token 0. engine and head as in greedy_decode."""
    if u.dim() != 2 or u.shape[1:] != prompt.shape[:1]:
        raise ValueError(f"u must be [steps, {prompt.shape[0]}]")

    def choose(logits, s):
        return sample(logits, u[s], temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)

    return _decode(model, prompt, u.shape[0], choose, graphed, engine, head)
