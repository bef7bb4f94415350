"""Rows near the ends of float32's range."""
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
