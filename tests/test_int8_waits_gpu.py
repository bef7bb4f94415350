"""The 8-bit product's bounded waits on a B200: a wait that gives up is reported, and leaves a context that works."""
import time

import pytest
import torch

from test_norm_kept_gpu import rows_of

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
TIMEOUT = 4  # FLB_ERR_TIMEOUT
LIMIT = 1 << 14  # polls of about 4 us, where a wait of a product is some microseconds


def product(x, w, out, step, limit=LIMIT, check=1):
    """flb_int8_linear_wait_test of x (Int8Rows, or a tensor) and w into out."""
    import flb_native as nat
    rows = not isinstance(x, torch.Tensor)
    (M, K), N = (x.codes if rows else x).shape, w.codes.shape[0]
    n = nat.lib.flb_int8_linear_workspace_bytes(M, N, K, int(rows))
    ws = nat.workspace(n, out.device)
    what = (None, 0, x.codes.data_ptr(), x.codes.stride(0), x.scale.data_ptr()) if rows else (x.data_ptr(), K, None, 0, None)
    return nat.lib.flb_int8_linear_wait_test(*what, w.codes.data_ptr(), w.codes.stride(0), w.scale.data_ptr(), None, 0, out.data_ptr(),
                                             M, N, K, nat.BF16, ws.data_ptr(), n, check, step, limit, nat.stream_of(out))


# the kernel for few tokens (K whole, and in parts), one block a tile, two blocks a tile; steps in the first ring and after it
CASES = [(40, 2048, 20000, 2), (40, 2048, 20000, 20), (100, 4096, 1000, 1), (2931, 768, 2304, 0), (2931, 768, 2304, 5),
         (2931, 768, 2304, 7), (5120, 1104, 2048, 0), (5120, 1104, 2048, 3), (5120, 1104, 2048, 11)]


def dropped(x, w, step):
    import flb_native as nat
    import kernels
    M, N = (x if isinstance(x, torch.Tensor) else x.codes).shape[0], w.codes.shape[0]
    want = kernels.int8_linear(x, w)
    out = torch.empty(M, N, dtype=BF, device="cuda")
    assert product(x, w, out, -1) == 0 and torch.equal(out, want)
    start = time.perf_counter()
    assert product(x, w, out, step) == TIMEOUT and b"gave up" in nat.lib.flb_last_error()
    took = time.perf_counter() - start
    torch.cuda.synchronize()
    assert took < 5, took  # every wait ended at its limit
    for _ in range(3):
        assert product(x, w, out, -1) == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M,K,N,step", CASES)
def test_a_lost_step_is_reported(M, K, N, step):
    import kernels
    x = kernels.quantize_int8(rows_of((M, K), BF, 1).cuda())
    w = kernels.quantize_int8(rows_of((N, K), BF, 2).cuda())
    dropped(x, w, step)


# the decoding step's kernel: one block a tile (several tiles each), clusters of two, four and eight
@pytest.mark.parametrize("M,K,N,step", [(1, 768, 32000, 3), (2, 768, 32000, 8), (3, 2000, 8190, 2), (7, 2048, 1000, 1), (4, 4096, 1000, 3)])
def test_a_lost_step_of_a_decoding_step_is_reported(M, K, N, step):
    import kernels
    x = rows_of((M, K), BF, 1).cuda()
    dropped(x, kernels.quantize_int8(rows_of((N, K), BF, 2).cuda()), step)


def late(rows, delay_us):
    """Rows whose codes and scales are copied into place after the delay, by kernels that let their successor start."""
    import flb_native as nat
    import kernels
    M, pitch = rows.codes.shape[0], rows.codes.stride(0)
    buffer = torch.zeros(M * pitch + 4 * M + 16, dtype=torch.uint8, device="cuda")
    source = torch.cat([rows.codes.as_strided((M * pitch,), (1,)).view(torch.uint8), rows.scale.view(torch.uint8)])
    n = source.numel() // 16 * 16
    buffer[n:source.numel()].copy_(source[n:])
    torch.cuda.synchronize()
    codes = buffer[:M * pitch].view(torch.int8).view(M, pitch)[:, :rows.codes.shape[1]]
    out = kernels.Int8Rows(codes, buffer[M * pitch:M * pitch + 4 * M].view(torch.float32), rows.dtype)
    assert nat.lib.flb_selftest_late_copy(source.data_ptr(), buffer.data_ptr(), n, delay_us, nat.stream_of(buffer)) == 0
    return out, source


@pytest.mark.parametrize("M,K,N", [(40, 256, 20000), (300, 64, 17000), (2931, 768, 2304), (5120, 1104, 2048)])
def test_a_late_predecessor_is_waited_for(M, K, N):
    """The kernel that makes the rows lets the product start and takes far longer than a wait's limit: the limit is for the
    product's own steps."""
    import kernels
    x, w = (kernels.quantize_int8(rows_of((n, K), BF, n).cuda()) for n in (M, N))
    want = kernels.int8_linear(x, w)
    out = torch.empty_like(want)
    for delay in (0, 50000):
        rows, source = late(x, delay)
        assert product(rows, w, out, -1, limit=1 << 10, check=0) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want), delay
        out.zero_()


def test_check_timeout_from_python():
    """The checked call gives the unchecked one's output, and is refused while a graph is captured, which goes on."""
    import kernels
    w = kernels.quantize_int8(rows_of((300, 640), BF, 1).cuda())
    for M in (1, 64, 600):
        x = rows_of((M, 640), BF, M).cuda()
        want = kernels.int8_linear(x, w)
        assert torch.equal(kernels.int8_linear(x, w, check_timeout=True), want)
        assert torch.equal(kernels.int8_linear(kernels.quantize_int8(x), w, check_timeout=True), want)
        assert torch.equal(kernels.Int8Linear(w, check_timeout=True)(x), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="stream capture"):
            kernels.int8_linear(x, w, check_timeout=True)
        got = kernels.int8_linear(x, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("M,K,N", [(40, 256, 20000), (2931, 768, 2304), (5120, 1104, 2048), (1, 768, 32000)])
def test_everything_a_late_predecessor_writes_is_read_after_it(M, K, N):
    """Scales, bias and a decoding step's x, written beside the product's start to where other values were read before."""
    import flb_native as nat
    import kernels
    x, wt = rows_of((M, K), BF, 1).cuda(), kernels.quantize_int8(rows_of((N, K), BF, 2).cuda())
    rows = kernels.quantize_int8(x)
    old = torch.cat([t.float().view(torch.uint8).reshape(-1) for t in (rows.scale, wt.scale, torch.zeros(N, device="cuda"))] +
                    [x.view(torch.uint8).reshape(-1)])
    new = old.clone()
    sizes = [4 * M, 4 * N, 4 * N, 2 * M * K]

    def parts(buffer):
        sx, sw, bias, xs = buffer[:sum(sizes)].split(sizes)
        return sx.view(torch.float32), sw.view(torch.float32), bias.view(torch.float32), xs.view(BF).view(M, K)

    pad = torch.zeros(-sum(sizes) % 16, dtype=torch.uint8, device="cuda")
    old, new = torch.cat([old, pad]), torch.cat([new, pad])
    for t, f in zip(parts(new), (2.0, 0.5, None, None)):
        t.mul_(f) if f else t.copy_(torch.randn(t.shape, device="cuda"))
    both = [b for b in (old, new)]
    step = M <= 16
    n = nat.lib.flb_int8_linear_workspace_bytes(M, N, K, int(not step))
    ws = nat.workspace(n, x.device)
    out = torch.empty(M, N, dtype=BF, device="cuda")
    buffer = old.clone()

    def call(buffer):
        sx, sw, bias, xs = parts(buffer)
        what = (xs.data_ptr(), K, None, 0, None) if step else (None, 0, rows.codes.data_ptr(), rows.codes.stride(0), sx.data_ptr())
        assert nat.lib.flb_int8_linear(*what, wt.codes.data_ptr(), wt.codes.stride(0), sw.data_ptr(), bias.data_ptr(), nat.F32,
                                       out.data_ptr(), M, N, K, nat.BF16, ws.data_ptr(), n, 0, nat.stream_of(out)) == 0

    want = []
    for b in both:
        call(b)
        want.append(out.clone())
    assert not torch.equal(*want)
    for i in range(10):
        call(buffer)  # what is there now has been read
        assert nat.lib.flb_selftest_late_copy(both[i % 2].data_ptr(), buffer.data_ptr(), buffer.numel(), 100, nat.stream_of(out)) == 0
        call(buffer)
        torch.cuda.synchronize()
        assert torch.equal(out, want[i % 2]), i
