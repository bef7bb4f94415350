"""A product whose waits give up: outputs that did not come are NaN, also where nobody asks for the error word."""
import pytest
import torch

from test_fp8_waits_gpu import BF, SHAPES, product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K,N,drops", SHAPES)
@pytest.mark.parametrize("from_codes", [False, True])
def test_what_did_not_come_is_nan(M, K, N, drops, from_codes, dtype):
    """Every output is either right to the bit or NaN, and some are NaN: no other number gets out."""
    import kernels
    g = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, K, generator=g).to(dtype).cuda(), kernels.quantize_fp8(torch.randn(N, K, generator=g).cuda())
    want = kernels.fp8_linear(x, w, check_timeout=True)
    assert torch.isfinite(want).all()
    for drop in drops:
        st, out = product(x, w, drop, 500, 0, from_codes)
        lost = torch.isnan(out)
        assert st == 0 and lost.any() and torch.equal(out[~lost], want[~lost]), drop
        assert torch.equal(kernels.fp8_linear(x, w), want)
