"""Plain forms and measured cases of three operators around a model's vocabulary head: its product, the choice of
a token from its logits, and the step of its weights.

fp8     kernels.fp8_linear: x @ weight.T + bias with both operands in 8-bit floating point (e4m3: 4 bits of exponent,
        3 of mantissa) and a power of two for each block of 128 along the summed axis. For inference the weight is kept
        so (kernels.quantize_fp8). For training it is a plain tensor, and the gradients of x and of the weight are such
        products too, of operands in blocks along their own summed axes.
sample  kernels.sample: a token for each row of logits from one given uniform number, after a temperature, with the
        top k, the smallest set of the probability p, and those of at least min_p of the largest probability.
adamw   kernels.AdamW: one step over all of a model's tensors, moments in 32 bits, or in 8 with a power of two
        for each block of 128, rounded up or down at random; the random numbers are a mix of element, step and seed.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BLOCK = 128


def listed():
    return [
        # the logits of one new token, from a head kept in 8 bits: latency, and the weight's bytes
        {"name": "fp8_token", "op": "fp8", "train": False, "rows": 1, "k": 768, "n": 32000, "type": "bf16", "wtype": "bf16"},
        # a projection for one new token of each of 16 sequences
        {"name": "fp8_batch", "op": "fp8", "train": False, "rows": 16, "k": 4096, "n": 4096, "type": "f16", "wtype": "f16"},
        # a ragged batch of prompts through a layer of odd width, all in 32 bits
        {"name": "fp8_ragged", "op": "fp8", "train": False, "rows": 2931, "k": 1001, "n": 2304, "type": "f32", "wtype": "f32"},
        # a training step of a small layer, nothing a multiple of anything
        {"name": "fp8_train_odd", "op": "fp8", "train": True, "rows": 1003, "k": 769, "n": 517, "type": "f16", "wtype": "f32"},
        # a training step of the vocabulary head over 16 prompts of 1024 tokens: three products
        {"name": "fp8_train_head", "op": "fp8", "train": True, "rows": 16384, "k": 768, "n": 32000, "type": "bf16", "wtype": "f32"},
        # the next token of one sequence, with the usual settings: latency alone
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 32000, "type": "bf16", "settings": "common", "temperature": 0.8, "top_k": 50, "top_p": 0.95,
         "min_p": 0.0},
        # 16 requests, each with settings of its own (one of them greedy, one with all of its tokens masked)
        {"name": "sample_requests", "op": "sample", "rows": 16, "vocab": 32000, "type": "f32", "settings": "rows", "temperature": 1.0, "top_k": 0, "top_p": 1.0,
         "min_p": 0.0},
        # many sequences at once, each one's smallest set of nine tenths of the probability
        {"name": "sample_nucleus", "op": "sample", "rows": 256, "vocab": 32000, "type": "bf16", "settings": "common", "temperature": 1.0, "top_k": 0, "top_p": 0.9,
         "min_p": 0.0},
        # a large vocabulary of odd size
        {"name": "sample_wide", "op": "sample", "rows": 64, "vocab": 131071, "type": "f32", "settings": "common", "temperature": 1.2, "top_k": 0, "top_p": 1.0,
         "min_p": 0.02},
        # a small model of odd width in 16 bits, moments in 8 bits: many small tensors
        {"name": "adamw_small", "op": "adamw", "layers": 3, "dim": 257, "vocab": 1003, "type": "bf16", "bits": 8},
        # the 12-layer model: 183 tensors, 106 million parameters
        {"name": "adamw_model", "op": "adamw", "layers": 12, "dim": 768, "vocab": 32000, "type": "f32", "bits": 32},
        # the same with its moments in 8 bits; the pass also reads them out, as a program does that looks at or converts them
        {"name": "adamw_model8", "op": "adamw", "layers": 12, "dim": 768, "vocab": 32000, "type": "f32", "bits": 8},
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["fp8", "fp8", "fp8", "sample", "sample", "adamw"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "fp8":
        train = rng.random() < 0.5
        k, n = _spread(rng, 33, 8192), _spread(rng, 16, 32000)
        if rng.random() < 0.6:
            k, n = -(-k // 16) * 16, -(-n // 8) * 8
        top = min(16384, int(1.3e11 / (k * n)), int(2.6e8 / n))
        rows = _spread(rng, 1, max(1, top if train or rng.random() < 0.6 else min(top, 64)))
        return {"op": op, "train": train, "rows": rows, "k": k, "n": n, "type": t, "wtype": rng.choice([t, "f32"])}
    if op == "sample":
        vocab = _spread(rng, 2, 200000)
        return {"op": op, "rows": _spread(rng, 1, max(1, min(512, (1 << 23) // vocab))), "vocab": vocab, "type": t, "settings": rng.choice(["common", "rows"]),
                "temperature": round(rng.uniform(0.3, 1.6), 2), "top_k": rng.choice([0, 0, _spread(rng, 1, 1000)]), "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 3)])}
    return {"op": op, "layers": _spread(rng, 1, 10), "dim": _spread(rng, 24, 768), "vocab": _spread(rng, 64, 20000), "type": t, "bits": rng.choice([8, 32])}


# ---- inputs --------------------------------------------------------------------------------------------------

def _shapes(case):
    """The tensors of an FLB model: two norms, two priors, two gates, q, k, v, the additive attention's vector and the output map a layer,
    and the embedding and the head."""
    d = case["dim"]
    layer = [(d,)] * 4 + [(d, d)] * 2 + [(d, d), (d,)] * 2 + [(d, d)] * 4 + [(d,)]
    return layer * case["layers"] + [(case["vocab"], d), (case["vocab"], d), (case["vocab"],)]


_ADAM = {"lr": 3e-4, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}
_STEP, _SEED = 1000, 12345   # steps already taken; the rounding's seed


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return (shift + scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "fp8":
        rows, k, n, wt = case["rows"], case["k"], case["n"], _TYPES[case["wtype"]]
        # a residual stream: tokens of their own spread, and a few channels far larger than the others
        loud = 1 + 15 * (uniform(k) < 0.01)
        s["x"] = (normal(rows, k, dtype=torch.float32) * torch.exp(0.5 * normal(rows, 1, dtype=torch.float32)) * loud).to(t)
        s["w"], s["b"] = normal(n, k, scale=1 / math.sqrt(k), dtype=wt), normal(n, scale=0.1, dtype=wt)
        if case["train"]:
            # gradients of a loss over tokens: small, some tokens' far larger than others'
            s["dy"] = (normal(rows, n, dtype=torch.float32) * torch.exp(normal(rows, 1, dtype=torch.float32)) / 64).to(t)
        else:
            s["wq"] = _fp8(s["w"].float())  # the weight as a program keeps it, in the plain form
    elif case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab, scale=2.0, dtype=torch.float32)
        # a few likely tokens over the others, and a tenth of them masked
        logits += torch.where(uniform(rows, vocab) < min(0.5, 20 / vocab), 6 * uniform(rows, vocab), 0)
        logits.masked_fill_(uniform(rows, vocab) < 0.1, -math.inf)
        s["u"] = uniform(rows)
        if case["settings"] == "rows":
            logits[rows // 2] = -math.inf
            s["temperature"] = 0.5 + uniform(rows)
            s["temperature"][0] = 0
            off = uniform(rows) < 0.3
            s["top_k"] = torch.where(off, 0, (1 + 100 * uniform(rows)).long())
            s["top_p"] = torch.where(uniform(rows) < 0.3, 1.0, 0.5 + 0.5 * uniform(rows))
            s["min_p"] = torch.where(uniform(rows) < 0.5, 0.0, 0.1 * uniform(rows))
        else:
            s.update({k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")})
        s["logits"] = logits.to(t)
    else:
        # All tensors in one buffer, each from a whole block of 128 on, as a program holds them that sends them over the network in one piece.
        # Gradients of each tensor's own size, moments as after many steps of such.
        shapes = _shapes(case)
        blocks = [-(-math.prod(x) // _BLOCK) for x in shapes]
        s["blocks"], s["shapes"] = blocks, shapes
        there = torch.cat([torch.arange(b * _BLOCK, device="cuda") < math.prod(x) for b, x in zip(blocks, shapes)]).view(-1, _BLOCK)
        scale = torch.cat([torch.full((b, 1), math.exp(i % 7 - 9), device="cuda") for i, b in enumerate(blocks)])
        s["p"] = normal(*there.shape, scale=0.02) * there
        s["g"] = (normal(*there.shape, dtype=torch.float32) * scale * there).to(t)
        m, v = 0.3 * s["g"].float().roll(1, 0) * there, scale * scale * (0.5 + uniform(*there.shape)) * there
        s["step"], s["taken"] = [torch.full((), _STEP, dtype=torch.int64, device="cuda") for _ in shapes], _STEP
        if case["bits"] == 8:
            noise = _noise(blocks, 0)
            (s["m"], s["me"]), (s["v"], s["ve"]) = _encode(m, noise >> 16, 14, 7, False), _encode(v, noise & 0xffff, 30, 8, True)
            s["m32"], s["v32"] = torch.zeros_like(m), torch.zeros_like(v)  # where the moments are read out to
        else:
            s["m"], s["v"] = m, v
    return s


# ---- the product, in 32 bits -----------------------------------------------------------------------------------

def _fp8(x):
    """What rows of float32 stand for in 8 bits: blocks of 128, each in units of the smallest power of two that keeps it within e4m3's 448."""
    v = torch.nn.functional.pad(x, (0, -x.shape[-1] % _BLOCK)).unflatten(-1, (-1, _BLOCK))
    top = v.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-127)
    half = torch.div(e, 2, rounding_mode="floor")  # in two steps: 2 ** 127 and its inverse
    codes = torch.ldexp(torch.ldexp(v, -half), half - e).to(torch.float8_e4m3fn).float()
    v = torch.where(torch.isfinite(top), torch.ldexp(torch.ldexp(codes, half), e - half), math.nan)
    return v.flatten(-2)[..., :x.shape[-1]]


def _plain_fp8(s):
    x, t, wt = s["x"].float(), s["x"].dtype, s["w"].dtype
    if not s["case"]["train"]:
        return (_fp8(x) @ s["wq"].t() + s["b"].float()).to(t)
    w, dy = s["w"].float(), s["dy"].float()
    y = _fp8(x) @ _fp8(w).t() + s["b"].float()
    dx = _fp8(dy) @ _fp8(w.t()).t()
    dw = _fp8(dy.t()) @ _fp8(x.t()).t()
    return y.to(t), dx.to(t), dw.to(wt), dy.sum(0).to(wt)


# ---- the choice of a token, in 64 bits: next to a border 32 would choose another one ---------------------------

def _settings(s):
    """Each setting as a column of 64-bit numbers."""
    rows = s["logits"].shape[0]
    return [(s[k].double() if torch.is_tensor(s[k]) else torch.full((rows,), float(s[k]), dtype=torch.float64, device="cuda"))[:, None]
            for k in ("temperature", "top_k", "top_p", "min_p")]


def _plain_sample(s):
    temperature, top_k, top_p, min_p = _settings(s)
    x = s["logits"].double()
    vocab = x.shape[1]
    # from the largest down, ties with the lowest index first
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    empty = x[:, :1] == -math.inf
    greedy = temperature <= 0
    w = torch.exp((x - torch.where(empty, 0, x[:, :1])) / torch.where(greedy, 1, temperature))
    rank = torch.arange(vocab, device="cuda")[None]
    w = torch.where((top_k <= 0) | (rank < top_k), w, 0)
    total = w.cumsum(1)
    w = torch.where(((total - w < top_p * total[:, -1:]) | (top_p >= 1) | (rank == 0)) & (w >= min_p), w, 0)
    # the first token, in the vocabulary's order, at which the sum passes u of the whole
    w = torch.zeros_like(w).scatter_(1, order, w)
    total = w.cumsum(1)
    token = (total <= s["u"].double()[:, None] * total[:, -1:]).sum(1)
    return torch.where(empty[:, 0], -1, torch.where(greedy[:, 0], order[:, 0], token))


# ---- the weights' step, in 32 bits -------------------------------------------------------------------------------

def _noise(blocks, step):
    """32 bits for each place of tensors of so many blocks: products with odd numbers (the digits of the golden ratio and of the roots of 2 and 3) and shifts."""
    i = torch.cat([torch.arange(b * _BLOCK, device="cuda") for b in blocks]).view(-1, _BLOCK)
    i = (i * 0x9E3779B9 + step * 0x6A09E667 + _SEED) & 0xffffffff
    i = ((i ^ (i >> 16)) * 0xBB67AE85) & 0xffffffff
    return i ^ (i >> 16)


def _encode(x, noise, below, bits, unsigned):
    """Blocks of float32 as codes of `bits` bits (three of mantissa, the others exponent, in binades from `below` under the block's largest to one over it; 0 for
    zero) and a byte a block. noise: 16 bits an element, which round up or down. A sign goes on top, or (unsigned) what is too small becomes the smallest."""
    raw = x.contiguous().view(torch.int32)
    size = raw & 0x7fffffff
    top = size.amax(1, keepdim=True) >> 23
    exps = torch.where(top == 255, 255, top.clamp(min=below + 1))
    key = torch.minimum((size + (noise.int() << 4)) >> 20, torch.tensor(254 * 8 + 7, device="cuda")) - ((exps - below) << 3)
    code = torch.where(key < 1, torch.where(size > 0, 1, 0) if unsigned else 0, torch.where(size > 0, key, 0))
    if not unsigned:
        code = code | torch.where(raw < 0, 1 << bits, 0)
    return code.to(torch.uint8), exps.to(torch.uint8).view(-1)


def _decode(codes, exps, below, bits):
    c, e = codes.int(), exps.int()[:, None]
    low = c & ((1 << bits) - 1)
    x = torch.where(low > 0, (low + ((e - below) << 3)) << 20, 0).view(torch.float32)
    return torch.where(e == 255, math.nan, torch.where(c > low, -x, x))


def _plain_adamw(s):
    (b1, b2), lr, eps, decay = _ADAM["betas"], _ADAM["lr"], _ADAM["eps"], _ADAM["weight_decay"]
    eight = s["case"]["bits"] == 8
    s["taken"] = step = s["taken"] + 1
    p, g = s["p"].float(), s["g"].float()
    m, v = (_decode(s["m"], s["me"], 14, 7), _decode(s["v"], s["ve"], 30, 8)) if eight else (s["m"], s["v"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    root = torch.sqrt(v) / math.sqrt(1 - b2 ** step) + eps
    # into the state's own tensors, as an optimizer's step
    s["p"].copy_(p * (1 - lr * decay) - lr / (1 - b1 ** step) * (m / root))
    if not eight:
        return s["p"], s["m"].copy_(m), s["v"].copy_(v)
    noise = _noise(s["blocks"], step)
    (s["m"], s["me"]), (s["v"], s["ve"]) = _encode(m, noise >> 16, 14, 7, False), _encode(v, noise & 0xffff, 30, 8, True)
    return s["p"], s["m32"].copy_(_decode(s["m"], s["me"], 14, 7)), s["v32"].copy_(_decode(s["v"], s["ve"], 30, 8))


def run(state):
    if own:
        return _own(state)
    return {"fp8": _plain_fp8, "sample": _plain_sample, "adamw": _plain_adamw}[state["case"]["op"]](state)


# ---- the framework's calls -----------------------------------------------------------------------------------

def _own(s):
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flb-transformer_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kernels

    c = s["case"]
    if c["op"] == "fp8" and not c["train"]:
        if "w8" not in s:
            s["w8"] = kernels.quantize_fp8(s["w"])  # once, as a program keeps it
        return kernels.fp8_linear(s["x"], s["w8"], s["b"])
    if c["op"] == "fp8":
        leaves = [s[k].requires_grad_(True) for k in ("x", "w", "b")]
        y = kernels.fp8_linear(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    if c["op"] == "sample":
        return kernels.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    eight = c["bits"] == 8
    if "adamw" not in s:
        # the optimizer that a program holds, its tensors' gradients, and the moments that it has by now
        def parts(x, shaped=True):
            whole = x.split(s["blocks"])
            return [y.view(-1)[:math.prod(z)].view(z) for y, z in zip(whole, s["shapes"])] if shaped else whole
        params = parts(s["p"])
        s["adamw"] = o = kernels.AdamW(params, **_ADAM, state_bits=c["bits"], seed=_SEED)
        for p, g, step, m, v in zip(params, parts(s["g"]), s["step"], parts(s["m"], not eight), parts(s["v"], not eight)):
            p.grad = g
            o.state[p] = {"step": step, "exp_avg": m, "exp_avg_sq": v}
        if eight:
            for p, m, v in zip(params, parts(s["me"], False), parts(s["ve"], False)):
                o.state[p].update(exp_avg_exps=m, exp_avg_sq_exps=v)
            s["out"] = list(zip(parts(s["m32"]), parts(s["v32"])))
    s["adamw"].step()
    if eight:
        s["adamw"].moments(out=s["out"])
    return s["p"], s["m32" if eight else "m"], s["v32" if eight else "v"]


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    e = 4 if case["type"] == "f32" else 2
    if case["op"] == "fp8":
        m, k, n, ew = case["rows"], case["k"], case["n"], 4 if case["wtype"] == "f32" else 2
        if not case["train"]:
            # x, the weight's codes with their powers of two, the bias; y
            return {"bytes": m * k * e + n * k + n * -(-k // _BLOCK) + n * ew + m * n * e, "flops": 2 * m * n * k}
        # x, dy, the weight and bias; y, dx, and the weight's and bias's gradients
        return {"bytes": 2 * m * k * e + 2 * m * n * e + 2 * (n * k + n) * ew, "flops": 6 * m * n * k}
    if case["op"] == "sample":
        r = case["rows"]
        return {"bytes": r * case["vocab"] * e + r * (4 + 8) + (20 * r if case["settings"] == "rows" else 0), "flops": 4 * r * case["vocab"]}
    n = sum(math.prod(x) for x in _shapes(case))
    # parameters and gradients in, parameters out; the moments in and out, and those of 8 bits read out in 32
    return {"bytes": n * 3 * e + (16 * n if case["bits"] == 32 else n * 12 + 4 * (n // _BLOCK)), "flops": 15 * n}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------

def _round8(x):
    """Along the last axis: units that bring the largest of each 128 to at most 448, then four bits of each value (fewer under 2 ** -6 units)."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], _BLOCK):
        part = x[..., at:at + _BLOCK]
        top = part.abs().amax(-1, keepdim=True)
        unit = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=-127))
        unit = torch.where(unit * 448 < top, unit * 2, torch.where((unit * 224 >= top) & (unit > 2.0 ** -127), unit / 2, unit))  # where log2 was a bit off
        q = part / unit
        fine = torch.exp2(torch.frexp(q)[1].clamp(min=-5).double() - 4)
        out[..., at:at + _BLOCK] = torch.round(q / fine) * fine * unit
    return out


def exact(case, seed):
    if case["op"] == "adamw":
        return _exact_adamw(prepare(case, seed))
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    x, w, b = (s[k].double() for k in ("x", "w", "b"))
    y = torch.matmul(_round8(x), _round8(w).transpose(0, 1)).add_(b)
    if not case["train"]:
        return y
    dy = s["dy"].double()
    dx = torch.matmul(_round8(dy), _round8(w.transpose(0, 1).contiguous()).transpose(0, 1))
    dw = torch.matmul(_round8(dy.transpose(0, 1).contiguous()), _round8(x.transpose(0, 1).contiguous()).transpose(0, 1))
    return y, dx, dw, torch.sum(dy, dim=0)


def _exact_sample(s):
    """Row by row: the tokens that may come are named by a threshold and how many may equal it."""
    out = []
    settings = [c[:, 0].tolist() for c in _settings(s)]
    for row, u, temperature, k, p, low in zip(s["logits"].double(), s["u"].tolist(), *settings):
        best = row.max()
        if best == -math.inf:
            out.append(-1)
        elif temperature <= 0:
            out.append(int((row == best).nonzero()[0]))
        else:
            kept = torch.argsort(-row, stable=True)
            kept = kept[:int(k)] if k > 0 else kept
            w = torch.exp((row[kept] - best) / temperature)
            if p < 1:
                before = torch.cat([w.new_zeros(1), w.cumsum(0)[:-1]])
                kept = kept[:max(1, int((before < p * w.sum()).sum()))]
            kept = torch.sort(kept)[0]
            w = torch.exp((row[kept] - best) / temperature)
            kept, w = kept[w >= low], w[w >= low]
            out.append(int(kept[torch.searchsorted(w.cumsum(0), u * w.sum(), right=True).clamp(max=len(kept) - 1)]))
    return torch.tensor(out, device=s["logits"].device)


def _exact_adamw(s):
    (b1, b2), step = _ADAM["betas"], _STEP + 1
    g, m, v = s["g"].double(), s["m"], s["v"]
    eight = s["case"]["bits"] == 8
    if eight:
        # by value: (1 + mantissa / 8) times the power of two that exponent field and block give
        def value(c, e, below, half):
            low, e = c.double() % half, e.double()[:, None]
            x = torch.where(low > 0, (1 + low % 8 / 8) * torch.exp2(torch.floor(low / 8) + e - below - 127), 0.0)
            return torch.where(c.double() >= half, -x, x)
        m, v = value(m, s["me"], 14, 128), value(v, s["ve"], 30, 256)
        # What is rounded to 8 bits are 32-bit numbers, whose last bit may decide: products and sums each rounded to 32 bits (of 64, which hold a product
        # of two such whole), by factors of 32 bits.
        r32 = lambda x: x.float().double()  # noqa: E731
        f = torch.tensor([b1, 1 - b1, b2, 1 - b2], device="cuda").double()
        m, v = r32(r32(m * f[0]) + r32(g * f[1])), r32(r32(v * f[2]) + r32(r32(g * g) * f[3]))
    else:
        m, v = b1 * m.double() + (1 - b1) * g, b2 * v.double() + (1 - b2) * g ** 2
    hat = m / (1 - b1 ** step) / (torch.sqrt(v / (1 - b2 ** step)) + _ADAM["eps"])
    p = s["p"].double() * (1 - _ADAM["lr"] * _ADAM["weight_decay"]) - _ADAM["lr"] * hat
    if eight:
        noise = _noise(s["blocks"], step).double()
        m, v = _exact_round(m, torch.floor(noise / 65536), 14, False), _exact_round(v, noise % 65536, 30, True)
    return p, m, v


def _exact_round(x, noise, below, unsigned):
    size = x.abs()
    top = size.amax(1, keepdim=True)
    top = torch.where(top > 0, (torch.frexp(top.float())[1].double() - 1).clamp(min=below - 126), below - 126.0)
    part, e = torch.frexp(size)
    r = torch.floor(16 * part + noise / 65536) * torch.exp2(e.double() - 4)
    least = torch.exp2(top - below) * 1.125
    r = torch.where(r < least, least if unsigned else 0.0, r)
    return torch.where(size > 0, torch.copysign(r, x), 0.0)
