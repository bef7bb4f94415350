"""The operators around a model's head at the sizes and mixtures of types from which they work in another way, against their
definitions: whole outputs, with the definitions evaluated in 64 bits on the GPU where they are large."""
import math

import pytest
import torch

from oracle import head as orc
from test_adamw_gpu import before, check as check_step
from test_fp8_linear_gpu import close, rows_of
from test_sample_gpu import LARGEST, logits_of

pytestmark = pytest.mark.gpu

BF, H, F = torch.bfloat16, torch.float16, torch.float32


def noise(at, n, t, seed):
    """orc.noise for the elements from `at` on, on the GPU."""
    i = torch.arange(at, at + n, device="cuda")
    x = (i * 0x9E3779B9 + t * 0x6A09E667 + seed) % 2 ** 32
    x = (x ^ (x >> 16)) * 0xBB67AE85 % 2 ** 32
    x = x ^ (x >> 16)
    return x >> 16, x & 0xffff


def values(s, name, at, n):
    """What the codes of a run of whole blocks stand for, float32."""
    below, unsigned = (14, False) if name == "exp_avg" else (30, True)
    blocks = slice(at // 128, -(-(at + n) // 128))
    return orc.moment_values(s[name][blocks], s[name + "_exps"][blocks], below, unsigned, n).float().cuda()


def check_run(opt, p, g, was, at, n, seed=0):
    """Elements at to at + n (whole blocks, or to the end) after a step: p, and the codes exactly. was: p, m and v of them, and the step."""
    group, s = opt.param_groups[0], opt.state[p]
    old, m, v, t = was
    t += 1
    g, got = g.view(-1)[at:at + n], p.detach().view(-1)[at:at + n].double()
    want, _, _, tol, _, _ = orc.adamw(old, g, m, v, t, group["lr"], group["betas"], group["eps"], group["weight_decay"])
    info = torch.finfo(p.dtype)
    assert ((got - want).abs() <= tol + info.eps / 2 * (want.abs() + tol) + info.smallest_normal * info.eps).all()
    m32, v32 = (x.cuda() for x in orc.moments32(g.cpu(), m.cpu(), v.cpu(), group["betas"]))
    rm, rv = noise(at, n, t, seed)
    blocks = slice(at // 128, -(-(at + n) // 128))
    for name, x, r, form in (("exp_avg", m32, rm, (14, False)), ("exp_avg_sq", v32, rv, (30, True))):
        codes, exps = orc.moment_codes(x, r, *form)
        assert torch.equal(s[name + "_exps"][blocks].long(), exps) and torch.equal(s[name][blocks].long(), codes), name


# Chunks of 8-bit moments are 4096 elements up to 24 for each SM, then 8192, 16384 and 32768: tensors that end within a step, within a chunk and with it.
@pytest.mark.parametrize("sizes", [(16_000_037, 1_053_443, 5), (20_000_003, 16_384, 11_000_123), (62_914_561, 98_304)], ids=str)
@pytest.mark.parametrize("dtype", [BF, F])
def test_adamw_codes_in_long_chunks(sizes, dtype):
    import kernels
    torch.manual_seed(len(sizes))
    params = [(0.1 * torch.randn(n, device="cuda")).to(dtype).requires_grad_(True) for n in sizes]
    opt = kernels.AdamW(params, lr=1e-2, state_bits=8, seed=3)
    for step in range(2):
        for p in params:
            p.grad = (0.01 * torch.randn(p.shape, device="cuda")).to(dtype)
        was = [p.detach().clone() for p in params]
        moments = opt.moments() if step else [(torch.zeros(p.shape, device="cuda"),) * 2 for p in params]
        opt.step()
        for p, old, (m, v) in zip(params, was, moments):
            check_run(opt, p, p.grad, (old, m, v, step), 0, p.numel(), seed=3)


def test_adamw_a_tensor_beyond_32_bits_of_offsets():
    import kernels
    n = 2 ** 31 + 128 * 77 + 3
    p = torch.zeros(n, dtype=BF, device="cuda").requires_grad_(True)
    p.grad = torch.empty(n, dtype=BF, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    opt = kernels.AdamW([p], lr=1e-2, state_bits=8)
    runs = [(0, 1 << 16), (2 ** 30 - 128 * 5, 1 << 16), (2 ** 31 - 128 * 64, n - (2 ** 31 - 128 * 64))]
    for step in range(2):
        was = []
        for at, k in runs:
            m, v = (values(opt.state[p], name, at, k) if step else torch.zeros(k, device="cuda") for name in ("exp_avg", "exp_avg_sq"))
            was.append((p.detach()[at:at + k].clone(), m, v, step))
        opt.step()
        for (at, k), w in zip(runs, was):
            check_run(opt, p, p.grad, w, at, k)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_parameters_of_three_types_in_a_group(bits):
    """A launch for each type, and each steps once."""
    import kernels
    g = torch.Generator().manual_seed(4)
    params = [(0.1 * torch.randn(s, generator=g)).to(t).cuda().requires_grad_(True)
              for s, t in (((300,), F), ((40, 7), BF), ((1000,), H), ((129,), BF), ((4097,), F), ((3, 5, 7), H))]
    opt = kernels.AdamW(params, lr=1e-2, state_bits=bits, seed=9)
    for _ in range(3):
        grads = [(0.01 * torch.randn(p.shape, generator=g)).to(p.dtype) for p in params]
        was = [before(opt, p, bits) for p in params]
        for p, x in zip(params, grads):
            p.grad = x.cuda()
        opt.step()
        for p, w, x in zip(params, was, grads):
            check_step(opt, p, w, x, bits, seed=9)


# More than 16 tiles of tokens, not a multiple of 16, with a weight that L2 does not keep (16 of them go through the channels together): by pairs of
# blocks, with an output that leaves L2 first; by one block, in parts of K
@pytest.mark.parametrize("M,K,N", [(4150, 6200, 8200), (2105, 130000, 400)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_fp8_tiles_of_tokens_in_groups(M, K, N, dtype):
    import kernels
    x, w = rows_of((M, K), dtype, M), rows_of((N, K), BF, N, 1 / math.sqrt(K))
    kept, xq = kernels.quantize_fp8(w.cuda()), kernels.quantize_fp8(x.cuda())
    got = kernels.fp8_linear(x.cuda(), kept, check_timeout=True)
    rows, cols = (torch.tensor([i for i in picks if i < n] + [n - 1]) for picks, n in (
        ((0, 1, 127, 128, 255, 256, 1000, 2047, 2048, 2100, 4095, 4096, 4100), M), ((0, 63, 64, 127, 128, 191, 192, 399, 4000, 8000, 8190), N)))
    close(got[rows][:, cols], *orc.fp8_product(x[rows], w[cols], None, dtype))
    # all of them, from the rows' values
    qx, qw = xq.dequantize().double(), kept.dequantize().double()
    want, size = qx @ qw.t(), qx.abs() @ qw.abs().t()
    tol = size * (min(K, 1024) / 32 * 2.0 ** -22 + math.ceil(K / 1024) * orc.EPS32)  # as in orc.fp8_product
    info = torch.finfo(dtype)
    tol += info.eps / 2 * (want.abs() + tol) + info.smallest_normal * info.eps / 2
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype,wtype", [(F, BF), (F, H), (BF, BF), (BF, H), (H, F)])
@pytest.mark.parametrize("M,K,N", [(130, 64, 1000), (1003, 769, 517)])
def test_fp8_gradients_of_other_types(M, K, N, dtype, wtype):
    import kernels
    x, w, b = rows_of((M, K), dtype, 1, 0.1), rows_of((N, K), wtype, 2, 1 / math.sqrt(K)), rows_of((N,), F, 3)
    dy = rows_of((M, N), dtype, 4, 0.01)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = kernels.fp8_linear(*leaves)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    assert (y.dtype, *(t.dtype for t in grads)) == (dtype, dtype, wtype, F)
    close(y, *orc.fp8_product(x, w, b, dtype), "y")
    close(grads[0], *orc.fp8_product(dy, w.t(), None, dtype), "dx")
    close(grads[1], *orc.fp8_product(dy.t(), x.t(), None, wtype), "dW")


@pytest.mark.parametrize("settings", [{}, {"top_p": 0.8}, {"top_k": 100, "top_p": 0.9}, {"top_k": 3000}, {"min_p": 0.01}, {"temperature": 0}], ids=str)
@pytest.mark.parametrize("dtype", [BF, H])
def test_sample_rows_that_shared_memory_does_not_hold(dtype, settings):
    """16-bit logits read from memory in each pass, at a pitch and from a start that are odd."""
    import kernels
    x, u = logits_of(80, LARGEST, dtype, 7)
    wide = torch.zeros(80, LARGEST + 7, dtype=dtype)
    wide[:, 3:LARGEST + 3] = x
    got = kernels.sample(wide.cuda()[:, 3:LARGEST + 3], u.cuda(), **settings).cpu()
    few = torch.tensor([0, 1, 2, 40, 79])
    assert got[few].tolist() == orc.sample(x[few], u[few], **settings).tolist()
    # and all rows as they come one at a time, by another number of blocks
    for r in (3, 17, 78):
        assert int(kernels.sample(x[r].cuda(), u[r].cuda(), **settings)) == int(got[r])
