"""Plain forms and measured cases of three families of operators.

norm   kernels.layer_norm: LayerNorm over the last axis, forward alone or forward and backward, with one
       weight for all rows or one per leading group (the wavefront's cells of one tick carry their layers'
       weights). With keep8 the backward reads its normalised rows from 8 bits.
gate   kernels.sigmoid_gate: x * sigmoid(z), forward and backward, x and z kept in 8 bits in between.
pack   kernels.pack8 and kernels.unpack8: a tensor into its 8-bit kept form and back.
int8   kernels.int8_linear: rows to 8-bit integers with a scale each, times 8-bit weight rows with a scale
       each; with norm the rows come from kernels.layer_norm_int8.

The kept form holds blocks of 128 consecutive elements of a row as integers of at most 127 in magnitude
times a power of two, the smallest for which the block's largest magnitude still rounds to at most 127.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-5
_BLOCK = 128


def listed():
    return [
        # one new token of each of 16 sequences through the model's 768-wide norm: latency alone
        {"name": "norm_token", "op": "norm", "train": False, "keep8": False, "groups": 1, "rows": 16, "dim": 768, "type": "bf16", "wtype": "f32"},
        # the normalised inputs of one wavefront tick: six cells, a weight each, 32 sequences
        {"name": "norm_tick", "op": "norm", "train": True, "keep8": False, "groups": 6, "rows": 32, "dim": 1024, "type": "f16", "wtype": "f32"},
        # a training step over 16 x 1024 tokens with no 16-byte row: odd rows, odd width, all in 32 bits
        {"name": "norm_odd", "op": "norm", "train": True, "keep8": False, "groups": 1, "rows": 16383, "dim": 1001, "type": "f32", "wtype": "f32"},
        # a large training batch, width 4096
        {"name": "norm_large", "op": "norm", "train": True, "keep8": False, "groups": 1, "rows": 32768, "dim": 4096, "type": "bf16", "wtype": "bf16"},
        # the same operator with its rows kept in 8 bits, at the model's width
        {"name": "norm_kept", "op": "norm", "train": True, "keep8": True, "groups": 1, "rows": 16384, "dim": 768, "type": "bf16", "wtype": "bf16"},
        # the gates of one tick and of a whole batch of tokens, x and z kept in 8 bits
        {"name": "gate_tick", "op": "gate", "rows": 96, "dim": 768, "type": "bf16"},
        {"name": "gate_kept", "op": "gate", "rows": 65536, "dim": 1024, "type": "bf16"},
        # any activation into its kept form and back: the q | k | v rows of three tokens a cell
        {"name": "pack_qkv", "op": "pack", "rows": 49152, "dim": 2304, "type": "bf16"},
        # vocabulary logits of one token, and of 16 sequences
        {"name": "int8_one", "op": "int8", "norm": False, "rows": 1, "k": 768, "n": 32000, "type": "bf16"},
        {"name": "int8_batch", "op": "int8", "norm": False, "rows": 16, "k": 4096, "n": 4096, "type": "f16"},
        # a norm and its projection to q | k | v over a ragged batch of prompts
        {"name": "int8_norm_qkv", "op": "int8", "norm": True, "rows": 2931, "k": 768, "n": 2304, "type": "bf16"},
        # every position's vocabulary logits: 16 prompts of 1024 tokens
        {"name": "int8_logits", "op": "int8", "norm": False, "rows": 16384, "k": 768, "n": 32000, "type": "bf16"},
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "kept", "gate", "pack", "int8", "int8"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "kept"):
        dim, groups = _spread(rng, 17, 8192), rng.choice([1, 1, 2, 7])
        if rng.random() < 0.6:
            dim = -(-dim // 8) * 8
        rows = _spread(rng, 1, min(32768, (1 << 27) // (dim * groups)))
        kept = op == "kept"
        if kept and t == "f32":
            t = "bf16"
        return {"op": "norm", "train": kept or rng.random() < 0.7, "keep8": kept, "groups": groups, "rows": rows, "dim": dim, "type": t,
                "wtype": t if kept else rng.choice([t, "f32"])}
    if op in ("gate", "pack"):
        dim = _spread(rng, 17, 8192)
        if rng.random() < 0.6:
            dim = -(-dim // 8) * 8
        return {"op": op, "rows": _spread(rng, 1, min(65536, (1 << 26) // dim)), "dim": dim, "type": t}
    k, n = _spread(rng, 33, 8192), _spread(rng, 16, 32000)
    if rng.random() < 0.7:
        k, n = -(-k // 16) * 16, -(-n // 8) * 8
    top = min(16384, int(4e11 / (k * n)), int(5.2e8 / n))
    rows = _spread(rng, 1, max(1, top if rng.random() < 0.6 else min(top, 64)))
    return {"op": "int8", "norm": rng.random() < 0.35, "rows": rows, "k": k, "n": n, "type": t}


def _activations(g, rows, dim, dtype):
    """Rows as a residual stream has them: each with its own spread and offset, and a few channels that are far larger than the others."""
    x = torch.randn(rows, dim, generator=g, device="cuda")
    spread = torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    loud = 1 + 15 * (torch.rand(dim, generator=g, device="cuda") < 0.01)
    return (x * spread * loud + 0.2 * torch.randn(rows, 1, generator=g, device="cuda")).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return (shift + scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)

    s = {"case": case}
    if case["op"] == "norm":
        groups, rows, dim, wt = case["groups"], case["rows"], case["dim"], _TYPES[case["wtype"]]
        lead, wlead = ((groups, rows), (groups,)) if groups > 1 else ((rows,), ())
        s["x"] = _activations(g, groups * rows, dim, t).reshape(*lead, dim)
        s["w"], s["b"] = normal(*wlead, dim, scale=0.2, shift=1.0, dtype=wt), normal(*wlead, dim, scale=0.1, dtype=wt)
        if case["train"]:
            s["dy"] = normal(*lead, dim)
            for k in ("x", "w", "b"):
                s[k].requires_grad_(True)
    elif case["op"] == "gate":
        s["x"] = _activations(g, case["rows"], case["dim"], t).requires_grad_(True)
        s["z"] = normal(case["rows"], case["dim"], scale=1.5).requires_grad_(True)
        s["dy"] = normal(case["rows"], case["dim"])
    elif case["op"] == "pack":
        s["x"] = _activations(g, case["rows"], case["dim"], t)
    else:
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = _activations(g, rows, k, t)
        if case["norm"]:
            s["w"], s["b"] = normal(k, scale=0.2, shift=1.0), normal(k, scale=0.1)
        # the weight as a program keeps it: 8-bit rows that start every 16 bytes, and a scale each
        weight = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        s["scale"] = weight.abs().amax(1) / 127
        s["codes"] = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device="cuda")[:, :k]
        s["codes"].copy_(torch.round(weight / s["scale"][:, None]))
        s["bias"] = normal(n, scale=0.1)
    return s


# ---- plain forms, in 32 bits ---------------------------------------------------------------------------------

def _kept(x):
    """What the kept form of x [..., dim] stands for. frexp and ldexp by whole numbers are exact, and so is the rounding."""
    dim = x.shape[-1]
    v = torch.nn.functional.pad(x, (0, -dim % _BLOCK)).unflatten(-1, (-1, _BLOCK))
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True))
    e = (e - 7 + (m >= 127.5 / 128).to(e.dtype)).clamp(min=-126)
    v = torch.ldexp(torch.round(torch.ldexp(v, -e)), e)
    return v.flatten(-2)[..., :dim]


def _rows8(x):
    """Codes (as floats) and scales of rows in 8-bit integers."""
    a = x.abs().amax(-1, keepdim=True)
    return torch.round(x * torch.where(a < 2.0 ** -118, torch.zeros_like(a), 127 / a)), a / 127


def _plain_norm(s):
    c, x, w, b = s["case"], s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    t, wt = s["x"].dtype, s["w"].dtype
    if c["groups"] > 1:
        w, b = w[:, None], b[:, None]
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
    h = centred * rstd
    y = (h * w + b).to(t)
    if not c["train"]:
        return y
    dy = s["dy"].float()
    if c["keep8"]:
        h = _kept(h)
    gw = dy * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    rows = 1 if c["groups"] > 1 else 0
    return y, dx.to(t), (dy * h).sum(rows).to(wt), dy.sum(rows).to(wt)


def _plain_gate(s):
    x, z, dy, t = s["x"].detach().float(), s["z"].detach().float(), s["dy"].float(), s["x"].dtype
    y = (x / (1 + torch.exp(-z))).to(t)
    x, gate = _kept(x), 1 / (1 + torch.exp(-_kept(z)))
    return y, (dy * gate).to(t), (dy * x * gate * (1 - gate)).to(t)


def _plain_int8(s):
    x, t = s["x"].float(), s["x"].dtype
    if s["case"]["norm"]:
        centred = x - x.mean(-1, keepdim=True)
        x = centred * torch.rsqrt((centred * centred).mean(-1, keepdim=True) + _EPS) * s["w"].float() + s["b"].float()
    q, scale = _rows8(x)
    return ((q @ s["codes"].float().t()) * scale * s["scale"] + s["bias"].float()).to(t)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        return _own(s, op)
    if op == "norm":
        return _plain_norm(s)
    if op == "gate":
        return _plain_gate(s)
    if op == "pack":
        return _kept(s["x"].float()).to(s["x"].dtype)
    return _plain_int8(s)


# ---- the framework's calls -----------------------------------------------------------------------------------

def _own(s, op):
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flb-transformer_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kernels

    c = s["case"]
    if op == "norm":
        if not c["train"]:
            return kernels.layer_norm(s["x"], s["w"], s["b"], eps=_EPS)
        y = kernels.layer_norm(s["x"], s["w"], s["b"], eps=_EPS, keep8=c["keep8"])
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"]))
    if op == "gate":
        y = kernels.sigmoid_gate(s["x"], s["z"], keep8=True)
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["z"]), s["dy"]))
    if op == "pack":
        return kernels.unpack8(kernels.pack8(s["x"]))
    weight = kernels.Int8Rows(s["codes"], s["scale"])
    x = kernels.layer_norm_int8(s["x"], s["w"], s["b"], eps=_EPS) if c["norm"] else s["x"]
    return kernels.int8_linear(x, weight, s["bias"])


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    e = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        ew = 4 if case["wtype"] == "f32" else 2
        n, d = case["groups"] * case["rows"] * case["dim"], case["groups"] * case["dim"]
        # x and y, and for training dy and dx; the weight and bias, and their gradients
        return {"bytes": (4 if case["train"] else 2) * n * e + (4 if case["train"] else 2) * d * ew, "flops": (19 if case["train"] else 8) * n}
    if case["op"] == "gate":
        n = case["rows"] * case["dim"]
        return {"bytes": 6 * n * e, "flops": 14 * n}
    if case["op"] == "pack":
        n = case["rows"] * case["dim"]
        return {"bytes": 2 * n * e, "flops": 4 * n}
    m, k, n = case["rows"], case["k"], case["n"]
    return {"bytes": m * k * e + n * k + n * 4 + n * e + m * n * e + (2 * k * e if case["norm"] else 0), "flops": 2 * m * n * k}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------

def _stands_for(x):
    """The kept form's values: per block the smallest power of two over (largest magnitude) / 127.5 as the unit."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], _BLOCK):
        part = x[..., at:at + _BLOCK]
        unit = torch.exp2(torch.frexp(part.abs().amax(-1, keepdim=True) / 127.5)[1].double().clamp(min=-126))
        out[..., at:at + _BLOCK] = torch.round(part / unit) * unit
    return out


def _normalised(x):
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    sigma = torch.sqrt(var + _EPS)
    return (x - mean) / sigma, sigma


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if k != "case"}
    if case["op"] == "norm":
        if case["groups"] > 1:
            d["w"], d["b"] = d["w"].unsqueeze(1), d["b"].unsqueeze(1)
        h, sigma = _normalised(d["x"])
        y = d["w"] * h + d["b"]
        if not case["train"]:
            return y
        if case["keep8"]:
            h = _stands_for(h)
        dh = d["dy"] * d["w"]
        n = case["dim"]
        along = (dh * h).sum(-1, keepdim=True) / n
        dx = (dh - dh.sum(-1, keepdim=True) / n - h * along) / sigma
        return y, dx, torch.sum(d["dy"] * h, dim=-2), torch.sum(d["dy"], dim=-2)
    if case["op"] == "gate":
        y = d["x"] * torch.sigmoid(d["z"])
        x, z = _stands_for(d["x"]), _stands_for(d["z"])
        return y, d["dy"] * torch.sigmoid(z), d["dy"] * x * torch.sigmoid(z) * torch.sigmoid(-z)
    if case["op"] == "pack":
        return _stands_for(d["x"])
    x = d["x"]
    if case["norm"]:
        x = _normalised(x)[0] * d["w"] + d["b"]
    unit = x.abs().max(dim=-1, keepdim=True).values / 127
    q = torch.round(x / unit.clamp(min=1e-300))
    return torch.matmul(q, d["codes"].transpose(0, 1)).mul_(unit).mul_(d["scale"]).add_(d["bias"])
