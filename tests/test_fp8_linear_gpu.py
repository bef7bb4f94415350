"""Products in 8-bit floating point on a B200, against their definition in 64 bits."""
import math

import pytest
import torch

from oracle import head as orc

pytestmark = pytest.mark.gpu

BF, H, F = torch.bfloat16, torch.float16, torch.float32


def rows_of(shape, dtype, seed, scale=1.0):
    """Rows of different sizes, with a few large columns."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(torch.randn(*shape[:-1], 1, generator=g))
    return (scale * x * (1 + 20 * (torch.rand(shape[-1], generator=g) < 0.02))).to(dtype)


def close(got, want, tol, what=""):
    got, nan = got.detach().double().cpu(), torch.isnan(want)
    assert got.shape == want.shape and torch.equal(torch.isnan(got), nan), what
    over = torch.where(nan, 0.0, (got - want).abs() - tol)
    assert (over <= 0).all(), (what, (torch.where(nan, 0.0, (got - want).abs()) / tol.clamp(min=1e-300)).max().item())


@pytest.mark.parametrize("K", [1, 3, 16, 31, 127, 128, 129, 512, 513, 768, 1001, 4096, 20000])
@pytest.mark.parametrize("dtype", [BF, H, F])
def test_rows_exact(K, dtype):
    import kernels
    x = rows_of((141, K), dtype, K)
    x[1] = 0
    x[2] = torch.finfo(dtype).max
    x[3] = torch.finfo(dtype).smallest_normal
    x[4, ::2] = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    x[5, K // 2], x[6, K - 1], x[7, 0] = math.inf, math.nan, -math.inf
    x[8], x[9], x[10] = 448, 449, -464
    x[11] = 1e-37 if dtype != H else 6e-8
    x[12, 0] = 3e4
    got = kernels.quantize_fp8(x.cuda())
    want, byte = orc.fp8_values(x)
    assert got.codes.shape == x.shape and got.codes.dtype == torch.float8_e4m3fn and got.dtype == dtype
    units = got.units().cpu()
    assert torch.equal(torch.isnan(units), byte == 255)
    assert torch.equal(torch.nan_to_num(units.double(), nan=0.0), torch.where(byte == 255, 0.0, torch.exp2(byte.double() - 127)))
    values = got.codes.float().cpu().double() * units.double().repeat_interleave(128, -1)[:, :K]
    assert torch.equal(torch.nan_to_num(values, nan=-1.0), torch.nan_to_num(want, nan=-1.0))
    small = torch.isfinite(want) & (want.abs() < 3e38)
    assert torch.equal(got.dequantize().cpu().double()[small], want[small])


# tokens around 8, 32 and a tile's 128; channels around a warp's 64 and a tile's 64, 128 and 192, ragged and odd; K around a block of 128, the four
# whose powers of two come together, an accumulator's 1024, parts of K
SHAPES = [(1, 768, 32000), (1, 1, 1), (2, 16, 8), (7, 128, 64), (9, 129, 65), (16, 4096, 4096), (17, 500, 130), (31, 1001, 257), (32, 512, 192), (33, 513, 193),
          (64, 16384, 64), (100, 640, 1000), (127, 1024, 384), (128, 1025, 129), (129, 768, 513), (257, 384, 4097), (300, 3000, 16), (700, 512, 1280),
          (2931, 768, 2304), (5000, 64, 640), (3, 32768, 40), (1000, 100, 8191), (260, 9000, 320), (4096, 2048, 1536), (130, 100, 20000)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F])
def test_product(M, K, N, dtype):
    import kernels
    x, w = rows_of((M, K), dtype, M + K), rows_of((N, K), BF, N, 1 / math.sqrt(K))
    bias = rows_of((N,), dtype, 5)
    want, tol = orc.fp8_product(x, w, bias, dtype)
    kept = kernels.quantize_fp8(w.cuda())
    got = kernels.fp8_linear(x.cuda(), kept, bias.cuda(), check_timeout=True)
    assert got.dtype == dtype
    close(got, want, tol)
    # from codes made before, from the plain weight, and again: the same bits
    assert torch.equal(kernels.fp8_linear(kernels.quantize_fp8(x.cuda()), kept, bias.cuda(), check_timeout=True), got)
    assert torch.equal(kernels.fp8_linear(x.cuda(), w.cuda(), bias.cuda()), got)
    for _ in range(3):
        assert torch.equal(kernels.fp8_linear(x.cuda(), kept, bias.cuda()), got)


@pytest.mark.parametrize("dtype,wtype,btype", [(H, H, None), (H, F, H), (BF, F, F), (F, BF, H), (F, F, None), (BF, H, BF)])
@pytest.mark.parametrize("M", [5, 140])
def test_types_and_bias(M, dtype, wtype, btype):
    import kernels
    x, w = rows_of((M, 300), dtype, 1, 0.1), rows_of((77, 300), wtype, 2, 0.05)
    bias = None if btype is None else rows_of((77,), btype, 3, 0.1)
    want, tol = orc.fp8_product(x, w, bias, dtype)
    close(kernels.fp8_linear(x.cuda(), kernels.quantize_fp8(w.cuda()), None if bias is None else bias.cuda()), want, tol)


# (tokens, K, channels): a token, ragged and odd ones, long sums over tokens in parts, the channels of a head
TRAIN = [(1, 1, 1), (1, 768, 2304), (3, 130, 5), (127, 129, 257), (130, 64, 1000), (1003, 769, 517), (4099, 257, 130), (2048, 768, 768), (700, 100, 8191), (20000, 64, 48)]


@pytest.mark.parametrize("M,K,N", TRAIN)
@pytest.mark.parametrize("dtype,wtype", [(BF, F), (F, F), (H, H)])
def test_gradients(M, K, N, dtype, wtype):
    import kernels
    x, w, b = rows_of((M, K), dtype, 1, 0.5), rows_of((N, K), wtype, 2, 1 / math.sqrt(K)), rows_of((N,), wtype, 3)
    dy = rows_of((M, N), dtype, 4, 0.1)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = kernels.fp8_linear(*leaves)
    grads = torch.autograd.grad(y, leaves, dy.cuda(), retain_graph=True)
    close(y, *orc.fp8_product(x, w, b, dtype), "y")
    close(grads[0], *orc.fp8_product(dy, w.t(), None, dtype), "dx")
    close(grads[1], *orc.fp8_product(dy.t(), x.t(), None, wtype), "dW")
    # sums in float32: of 128 tokens as four runs of 32, the tiles' in eight runs: every addition half a step of the magnitudes' sum
    total, size, info = dy.double().sum(0), dy.double().abs().sum(0), torch.finfo(wtype)
    additions = 34 + math.ceil(math.ceil(M / 128) / 8) + 8
    tol = size * additions * orc.EPS32
    close(grads[2], total, tol + info.eps / 2 * (total.abs() + tol) + info.smallest_normal * info.eps / 2, "db")
    for a, c in zip(grads, torch.autograd.grad(y, leaves, dy.cuda())):
        assert torch.equal(a, c)


def test_gradients_against_differences():
    """Small whole numbers are exact in 8 bits, and so are the products: the map's differences are its gradients, to the last bit."""
    import kernels
    g = torch.Generator().manual_seed(6)
    x, w, dy = (torch.randint(-7, 8, s, generator=g).float().cuda() for s in ((200, 150), (90, 150), (200, 90)))
    b = torch.zeros(90, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(kernels.fp8_linear(*leaves), leaves, dy)
    for i, t in enumerate((x, w, b)):
        d = torch.randint(-1, 2, t.shape, generator=g).float().cuda()
        args = [x, w, b]
        plus, minus = ([*args[:i], t + s * d, *args[i + 1:]] for s in (1, -1))
        difference = ((kernels.fp8_linear(*plus) - kernels.fp8_linear(*minus)).double() * dy.double()).sum() / 2
        assert difference == (grads[i].double() * d.double()).sum()


def test_gradients_that_are_asked_for():
    import kernels
    x, w, b = (rows_of(s, F, 7).cuda() for s in ((300, 140), (70, 140), (70,)))
    dy = rows_of((300, 70), F, 8).cuda()
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    all_three = torch.autograd.grad(kernels.fp8_linear(*full), full, dy)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2), (0, 1)):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(kernels.fp8_linear(*leaves), [leaves[i] for i in wanted], dy)
        for i, t in zip(wanted, got):
            assert torch.equal(t, all_three[i])
    # without a bias, leading axes, a gradient that is one number for all
    leaves = [t.clone().requires_grad_(True) for t in (x.view(3, 100, 140), w)]
    y = kernels.fp8_linear(*leaves)
    y.sum().backward()
    assert y.shape == (3, 100, 70) and leaves[0].grad.shape == (3, 100, 140)
    close(leaves[1].grad, *orc.fp8_product(torch.ones(70, 300), x.cpu().t(), None, F))
    with pytest.raises(RuntimeError, match="differentiable once"):
        z = torch.autograd.grad(kernels.fp8_linear(*full).sum(), full[0], create_graph=True)[0]
        z.sum().backward()


def test_infinities_stay_in_their_rows():
    import kernels
    x, w = rows_of((200, 300), BF, 9), rows_of((150, 300), BF, 10)
    x[3, 7], x[140, 299], w[20, 5] = math.inf, math.nan, -math.inf
    want, tol = orc.fp8_product(x, w, None, BF)
    assert torch.isnan(want).any(1).all() and torch.isnan(want[3]).all()
    close(kernels.fp8_linear(x.cuda(), kernels.quantize_fp8(w.cuda())), want, tol)


def test_small_and_large_units():
    """Blocks whose powers of two are far apart, and products near both ends of float32."""
    import kernels
    x, w = rows_of((40, 600), F, 11), rows_of((30, 600), F, 12)
    x[:, 128:256] *= 1e-12
    x[:, 256:384] *= 1e10
    x[7] *= 1e-30
    w[:, 256:384] *= 1e-18
    w[9] *= 1e20
    want, tol = orc.fp8_product(x, w, None, F)
    close(kernels.fp8_linear(x.cuda(), kernels.quantize_fp8(w.cuda())), want, tol)


def test_long_sums_are_rounded():
    """Over 65536 of K the error stays that of float32 sums (rms, relative to the results): accumulators of 1024 of K at most 32 steps of 2^-24 on
    average of a partial sum's size, about half of the result's growing as its root: 1e-6 is above that for each of 64 independent ones, and
    below what one accumulator would lose."""
    import kernels
    x, w = torch.randn(32, 65536, generator=torch.Generator().manual_seed(13)), torch.randn(96, 65536, generator=torch.Generator().manual_seed(14))
    want, _ = orc.fp8_product(x, w, None, F)
    got = kernels.fp8_linear(x.cuda(), kernels.quantize_fp8(w.cuda())).double().cpu()
    assert ((got - want).pow(2).mean().sqrt() / want.pow(2).mean().sqrt()) < 1e-6


def test_layouts():
    import kernels
    x, w = rows_of((60, 300), BF, 15), rows_of((90, 300), BF, 16)
    kept = kernels.quantize_fp8(w.cuda())
    want = kernels.fp8_linear(x.cuda(), kept)
    wide = torch.zeros(60, 3, 303, dtype=BF)
    wide[:, 1, 2:302] = x
    assert torch.equal(kernels.fp8_linear(wide.cuda()[:, 1, 2:302], kept), want)
    assert torch.equal(kernels.fp8_linear(x.t().contiguous().cuda().t(), kept), want)
    assert torch.equal(kernels.fp8_linear(x.view(3, 4, 5, 300).cuda(), kept), want.view(3, 4, 5, 90))
    assert torch.equal(kernels.fp8_linear(x[0].cuda(), kept), kernels.fp8_linear(x[:1].cuda(), kept)[0])
    assert torch.equal(kernels.fp8_linear(x.cuda(), w.t().contiguous().cuda().t()), want)
    # codes that do not start on 16 bytes are copied
    odd = kernels.Fp8Rows(kept.codes.contiguous(), kept.exps, kept.dtype)
    assert torch.equal(kernels.fp8_linear(x.cuda(), odd), want)
    # rows behind the last one are left as they were
    out = kernels.fp8_linear(x[:0].cuda(), kept)
    assert out.shape == (0, 90)
    none = kernels.quantize_fp8(w[:0].cuda())
    assert kernels.fp8_linear(x.cuda(), none).shape == (60, 0)
    for M, N in ((0, 90), (60, 0)):
        leaves = [x[:M].cuda().requires_grad_(True), w[:N].float().cuda().requires_grad_(True), torch.zeros(N, device="cuda", requires_grad=True)]
        kernels.fp8_linear(*leaves).sum().backward()
        assert all((t.grad == 0).all() and t.grad.shape == t.shape for t in leaves)


def test_captured_and_on_another_stream():
    """Forward and backward captured, twice, and replayed one after the other. (No eager graph of the same leaves may live then: torch's engine ties a
    leaf's gradient to the stream of its oldest graph, and refuses the capture, whatever the operator.)"""
    import kernels
    x, w, b = (rows_of(s, F, 17).cuda().requires_grad_(True) for s in ((130, 260), (70, 260), (70,)))
    dy = rows_of((130, 70), F, 18).cuda()
    eager = kernels.fp8_linear(x, w, b)
    want = torch.autograd.grad(eager, (x, w, b), dy)
    eager = eager.detach()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(kernels.fp8_linear(x, w, b), (x, w, b), dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = kernels.fp8_linear(x, w, b)
            outs.append((y, *torch.autograd.grad(y, (x, w, b), dy)))
        graphs.append(graph)
    kept = kernels.quantize_fp8(w.detach())
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            kernels.fp8_linear(x.detach(), kept, check_timeout=True)
    for graph in (*graphs, *graphs[::-1]):
        graph.replay()
    for out in outs:
        assert torch.equal(out[0], eager) and all(torch.equal(a, c) for a, c in zip(out[1:], want))


def test_modules():
    import kernels
    linear = torch.nn.Linear(100, 40).cuda()
    m = kernels.Fp8Linear.from_linear(linear)
    assert m.weight is linear.weight and m.bias is linear.bias and set(m.state_dict()) == {"weight", "bias"}
    x = torch.randn(7, 100, device="cuda")
    y = m(x)
    y.sum().backward()
    assert linear.weight.grad is not None
    kept = m.kept()
    assert torch.equal(kept(x), y) and not kept(x).requires_grad
    with torch.no_grad():
        m.weight += 1
    assert torch.equal(kept(x), y)
    for cast in (lambda t: t.to(BF), lambda t: t.half(), lambda t: t.double()):
        c = torch.nn.Sequential(m.kept())
        codes, exps = c[0].codes, c[0].exps
        cast(c)
        assert c[0].codes.dtype == torch.float8_e4m3fn and torch.equal(c[0].codes.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(c[0].exps, exps)
    assert torch.equal(m.kept().cpu().cuda()(x), m(x))
