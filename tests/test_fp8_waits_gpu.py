"""The waits of the 8-bit floating-point product that give up: reported, with nothing left in flight and the context usable."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def product(x, w, drop, limit, check, from_codes):
    """flb_fp8_linear_wait_test's status and output."""
    import flb_native as nat
    import kernels
    M, K = x.shape
    N = w.codes.shape[0]
    out = torch.empty(M, N, dtype=x.dtype, device="cuda")
    need = nat.lib.flb_fp8_linear_workspace_bytes(M, N, K, int(from_codes))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    xq = kernels.quantize_fp8(x)
    st = nat.lib.flb_fp8_linear_wait_test(None if from_codes else x.data_ptr(), K, xq.codes.data_ptr() if from_codes else None, xq.codes.stride(0),
                                          xq.exps.data_ptr() if from_codes else None, w.codes.data_ptr(), w.codes.stride(0), w.exps.data_ptr(), None, 0,
                                          out.data_ptr(), M, N, K, nat.dtype_code(x.dtype), ws.data_ptr(), need, check, drop, limit, nat.stream_of(x))
    return st, out


# one block a tile with 64 and 128 channels, pairs of blocks with one tile and several; K in parts. Steps that the first worker has: in the
# first ring and, where it has more, after it.
SHAPES = [(5, 768, 640, (0, 1, 4, 5)), (64, 768, 8000, (0, 3, 4)), (1500, 640, 2304, (0, 4)), (64, 4096, 512, (0, 1)), (2931, 1024, 2304, (0, 2, 5, 9))]


@pytest.mark.parametrize("M,K,N,drops", SHAPES)
@pytest.mark.parametrize("from_codes", [False, True])
def test_a_step_that_never_loads_is_reported(M, K, N, drops, from_codes):
    import kernels
    g = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, K, generator=g).to(BF).cuda(), kernels.quantize_fp8(torch.randn(N, K, generator=g).cuda())
    want = kernels.fp8_linear(x, w, check_timeout=True)
    for drop in drops:
        st, _ = product(x, w, drop, 500, 1, from_codes)
        assert st == 4, (drop, st)
        assert torch.equal(kernels.fp8_linear(x, w, check_timeout=True), want)
    st, out = product(x, w, -1, 1 << 20, 1, from_codes)
    assert st == 0 and torch.equal(out, want)
    # a step that there is not is not waited for
    st, out = product(x, w, 1 << 30, 1 << 20, 1, from_codes)
    assert st == 0 and torch.equal(out, want)


def test_behind_a_predecessor_that_ends_late():
    """The product's waits count its own steps alone, and it reads what a predecessor that lets it start early writes at its end."""
    import ctypes
    import flb_native as nat
    import kernels
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(40, 1024, generator=g).to(BF).cuda(), kernels.quantize_fp8(torch.randn(512, 1024, generator=g).cuda())
    want = kernels.fp8_linear(x, w)
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    nat.check(nat.lib.flb_selftest_late_copy(x.data_ptr(), late.data_ptr(), x.numel() * 2, 20000, ctypes.c_void_p(nat.stream_of(x))), "late copy")
    assert torch.equal(kernels.fp8_linear(late, w, check_timeout=True), want)
