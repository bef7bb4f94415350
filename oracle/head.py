"""Definitions, in 64 bits, of the operators around a model's head: the choice of a token from logits, AdamW's step with moments
in 32 or 8 bits. Plain loops and comparisons, on the CPU; bounds for float32 arithmetic beside the values."""
import math

import torch

EPS32 = 2.0 ** -24  # half a step of float32, relative


def kept_tokens(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The tokens of one row that may come, in the vocabulary's order, and their weights (float64). None: no token may."""
    x = logits.double()
    best = x.max()
    if torch.isnan(x).any() or best == -math.inf:
        return None
    if not temperature > 0:
        return torch.argmax((x == best).int())[None], torch.ones(1, dtype=torch.float64)
    ranked = torch.argsort(-x, stable=True)[:int((x > -math.inf).sum())]
    w = (x == best).double() if best == math.inf else torch.exp((x - best) / temperature)
    if 0 < top_k < len(ranked):
        ranked = ranked[:top_k]
    if top_p < 1:
        each = w[ranked]
        before = torch.cat([each.new_zeros(1), each.cumsum(0)[:-1]])
        kept = before < top_p * each.sum()
        kept[0] = True
        ranked = ranked[kept]
    ranked = torch.sort(ranked[w[ranked] >= min(min_p, 1.0)])[0]
    return ranked, w[ranked]


def sample(logits, u, **settings):
    """The token of each row of [rows, V]; a setting is a number or a list of one a row."""
    out = []
    for r, row in enumerate(logits):
        kept = kept_tokens(row, **{k: (v[r] if isinstance(v, (list, tuple)) else v) for k, v in settings.items()})
        if kept is None:
            out.append(-1)
            continue
        tokens, w = kept
        total = w.cumsum(0)
        over = (total > float(u[r]) * total[-1]).nonzero()
        out.append(int(tokens[over[0, 0]]) if len(over) else int(tokens[-1]))
    return torch.tensor(out)


# ---- AdamW ----------------------------------------------------------------------------------------------------

def adamw(p, g, m, v, t, lr, betas, eps, decay):
    """The step's p, m and v in float64 from what the inputs hold, and how far float32 arithmetic may take each (before p's own rounding)."""
    b1, b2 = betas
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m_new, v_new = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    # products with a rounded factor and their sum: 3 half steps of each product, one of the sum; g * g has one more
    tol_m = 4 * EPS32 * ((b1 * m).abs() + ((1 - b1) * g).abs())
    tol_v = 5 * EPS32 * v_new
    root = torch.sqrt(v_new / (1 - b2 ** t)) + eps
    step = lr / (1 - b1 ** t) * m_new / root
    # rate, root of v, its factor, the sum with eps and the division: approximate root and quotient within 2 steps (4 half steps) each
    tol_p = lr / (1 - b1 ** t) * tol_m / root + step.abs() * 16 * EPS32
    p_new = p * (1 - lr * decay) - step
    # the factor of p, and the last sum
    return p_new, m_new, v_new, tol_p + 2 * EPS32 * (p.abs() + p_new.abs()), tol_m, tol_v


def noise(n, t, seed):
    """16 bits for m and 16 for v of each element."""
    i = torch.arange(n, dtype=torch.int64)
    x = (i * 0x9E3779B9 + t * 0x6A09E667 + seed) % 2 ** 32
    x = (x ^ (x >> 16)) * 0xBB67AE85 % 2 ** 32
    x = x ^ (x >> 16)
    return x >> 16, x & 0xffff


def moment_codes(x, bits16, below, unsigned):
    """Codes [blocks, 128] and exponents [blocks] of a float32 moment, by integers one element at a time's rules."""
    n = x.numel()
    raw = torch.nn.functional.pad(x.reshape(-1), (0, -n % 128)).view(torch.int32).long() & 0xffffffff
    r = torch.nn.functional.pad(bits16, (0, -n % 128)).view(-1, 128)
    raw = raw.view(-1, 128)
    size = raw & 0x7fffffff
    top = size.amax(1, keepdim=True) >> 23
    e = torch.where(top == 255, 255, torch.clamp(top, min=below + 1))
    c = torch.clamp((size + r * 16) >> 20, max=254 * 8 + 7) - (e - below) * 8
    c = torch.where(size == 0, 0, torch.clamp(c, min=1 if unsigned else 0))
    if not unsigned:
        c = c + torch.where(raw >> 31 == 1, 128, 0)
    return c, e[:, 0]


def moment_values(codes, exps, below, unsigned, n):
    """What codes stand for, in float64."""
    c, e = codes.long().cpu().view(-1, 128), exps.long().cpu()[:, None]
    low = c if unsigned else c & 127
    x = torch.where(low > 0, (1 + low % 8 / 8) * torch.exp2((low // 8 + e - below - 127).double()), 0.0).double()
    x = torch.where((c > low), -x, x)
    return torch.where(e == 255, math.nan, x).reshape(-1)[:n]


def moments32(g, m, v, betas):
    """The new moments as products and sums rounded to float32 one by one (IEEE, on the CPU): what is rounded to 8 bits."""
    g, m, v = (x.float() for x in (g, m, v))
    f = [torch.tensor(x, dtype=torch.float64).float() for x in (betas[0], 1 - betas[0], betas[1], 1 - betas[1])]
    return m * f[0] + g * f[1], v * f[2] + (g * g) * f[3]


# ---- 8-bit floating point ---------------------------------------------------------------------------------------

def fp8_values(x):
    """What rows of [..., K] stand for in e4m3 with a power of two for each block of 128 (float64), and the blocks' powers of two as bytes."""
    x = x.double()
    K = x.shape[-1]
    blocks = torch.nn.functional.pad(x, (0, -K % 128)).unflatten(-1, (-1, 128))
    top = blocks.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    byte = torch.zeros(top.shape, dtype=torch.int64)
    for b in range(254, -1, -1):  # the smallest unit in which the largest is at most 448
        byte = torch.where(fine & (top <= 448 * 2.0 ** (b - 127)), b, byte)
    q = torch.where(fine, blocks, 0) / torch.exp2((byte - 127).double())
    # to 4 significant bits, or multiples of 2^-9 below 2^-6
    e = torch.clamp(torch.frexp(q)[1] - 4, min=-9)
    step = torch.exp2(e.double())
    q = torch.round(q / step) * step * torch.exp2((byte - 127).double())
    q = torch.where(fine, q, math.nan)
    return q.flatten(-2)[..., :K], torch.where(fine, byte, 255)[..., 0]


def fp8_product(x, w, bias, dtype):
    """x [M, K] times w [N, K] rows, both as their 8-bit values: float64, and how far a result of `dtype` may be.

    Each step of 32 of K that the tensor core adds to an accumulator of 1024 is taken to lose at most 2^-22 of the sum S of the
    magnitudes so far: 32 such of each accumulator's own S. Accumulators are added in float32, half a step each, and the bias; then the output's
    own rounding."""
    qx, qw = fp8_values(x)[0], fp8_values(w)[0]
    y, size = qx @ qw.t(), qx.abs() @ qw.abs().t()
    K = x.shape[1]
    tol = size * (min(K, 1024) / 32 * 2.0 ** -22 + math.ceil(K / 1024) * EPS32)
    if bias is not None:
        y = y + bias.double()
        tol = tol + EPS32 * (y.abs() + bias.double().abs())
    info = torch.finfo(dtype)
    return y, tol + info.eps / 2 * (y.abs() + tol) + info.smallest_normal * info.eps / 2
