"""Rows near the ends of float32's range: LayerNorm and its kept form, the kept form's errors, integer products."""
import pytest
import torch

from oracle import rows as orc
from test_norm_kept_gpu import close, cuda, params, rows_of

pytestmark = pytest.mark.gpu

BF, H, F = torch.bfloat16, torch.float16, torch.float32

# widths that leave lanes of a warp's last chunk empty, or none; in every mode and layout
WIDTHS = [20, 24, 256, 300, 600, 1001, 2056, 8200]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, F])
def test_norm_of_large_constant_rows(D, dtype):
    """Rows of 2^110 throughout: sums and mean are exact, h is zero and 1/sigma is 1 / sqrt(eps), a million here. A lane beyond
    the row must not count as an element of value zero, whose h would be infinite."""
    import kernels
    x = torch.full((5, D), 2.0 ** 110).to(dtype)
    x[3] = rows_of((D,), dtype, 3)
    (w, b), dy, eps = params((D,), F, 1), rows_of((5, D), dtype, 2), 1e-12
    leaves = [t.requires_grad_(True) for t in cuda(x, w, b)]
    y = kernels.layer_norm(*leaves, eps=eps)
    got = torch.autograd.grad(y, leaves, dy.cuda())
    _, _, (h, rs, dh) = orc.layer_norm(x, w, b, eps, dtype)
    flat = [0, 1, 2, 4]
    h, dh = h.clone(), dh.clone()
    assert not h[flat].any()
    dh[flat] = 0  # exact
    for g, (v, tol), name in zip(got, orc.layer_norm_backward(h, rs, dh, w, dy, dtype, F), ("dx", "dw", "db")):
        close(g, v, tol, name)


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, F])
def test_norm_of_rows_whose_sum_overflows(D, dtype):
    """The mean of such a row is infinite: its outputs are NaN, and what is kept of it in 8 bits is NaN throughout, so that its
    gradient is, kept or not. Other rows are as ever."""
    import kernels
    x, (w, b), dy = rows_of((6, D), dtype, D), params((D,), F, 1), rows_of((6, D), dtype, 2)
    x[1], x[4] = 3e38, -3e38
    fine = [0, 2, 3, 5]
    want, tol, _ = orc.layer_norm(x[fine], w, b, 1e-5, dtype)
    for keep8 in (False, True):
        xs, ws, bs = cuda(x, w, b)
        xs.requires_grad_(True)
        y = kernels.layer_norm(xs, ws, bs, keep8=keep8)
        close(y[fine], want, tol, "y")
        (dx,) = torch.autograd.grad(y, xs, dy.cuda())
        for t in (y, dx):
            assert torch.isnan(t[[1, 4]]).all() and torch.isfinite(t[fine]).all(), keep8


@pytest.mark.parametrize("dtype", [BF, F])
def test_kept_errors_over_the_range(dtype):
    """What the kept form is off by: 1/127 of the block's largest magnitude between the ends of the range, 2^-127 below
    them, and one unit in 63 where the largest magnitude would round to 64 * 2^122, which float32 does not hold."""
    import kernels
    g = torch.Generator().manual_seed(0)
    x = torch.randn(400, 128, generator=g, dtype=torch.float64)
    x = x / x.abs().amax(-1, keepdim=True) * torch.exp2(torch.linspace(-140, 128, 400, dtype=torch.float64)[:, None])
    x = torch.cat([x, torch.full((1, 128), torch.finfo(dtype).max, dtype=torch.float64)])
    x = x.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)
    got = kernels.unpack8(kernels.pack8(x.cuda()), F).cpu().double()
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    bound = torch.maximum(top / 127, torch.full_like(top, 2.0 ** -127))
    bound = torch.where(top >= 63.5 * 2.0 ** 122, top / 63, bound)
    assert ((got - x).abs() <= bound).all()
    assert not got[top[:, 0] < 2.0 ** -127].any()


# the kernels of a decoding step (alone, in clusters), of few tokens (whole and partial tiles, K in parts), of many tokens,
# and of two blocks a tile
@pytest.mark.parametrize("M,K,N", [(1, 768, 32000), (3, 2048, 300), (20, 256, 20000), (20, 4096, 300), (300, 64, 17000), (2931, 768, 2304),
                                   (2600, 1056, 4104)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_products_of_large_rows(M, K, N, dtype):
    """An integer sum times a token's scale alone can pass float32 where the output does not."""
    import kernels
    x = rows_of((M, K), F, 1)
    x[::2] *= 3e36
    x = x.to(dtype)
    wt = kernels.quantize_int8((rows_of((N, K), F, 2) * 1e-6).cuda())
    bias = params((N,), dtype, 3)[1]
    want, tol = orc.int8_product(*orc.int8_rows(x), wt.codes.cpu(), wt.scale.cpu(), bias, dtype)
    assert want.abs().max() < 1e35
    rows = kernels.quantize_int8(x.cuda())
    assert rows.scale.max() > 1e35
    close(kernels.int8_linear(x.cuda(), wt, bias.cuda()), want, tol, "from x")
    close(kernels.int8_linear(rows, wt, bias.cuda()), want, tol, "from rows")
