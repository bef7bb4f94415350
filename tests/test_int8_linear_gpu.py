"""8-bit integer rows and their product on a B200, against exact integer sums in 64 bits."""
import math

import pytest
import torch

from oracle import rows as orc
from test_norm_kept_gpu import close, cuda, params, rows_of

pytestmark = pytest.mark.gpu

BF, H, F = torch.bfloat16, torch.float16, torch.float32


def weight(N, K, seed):
    """A weight's codes and scales on the CPU, and as the operator takes them."""
    import kernels
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(seed)) / math.sqrt(K)
    q = kernels.quantize_int8(w.cuda())
    return q.codes.cpu(), q.scale.cpu(), q


@pytest.mark.parametrize("K", [1, 3, 16, 31, 127, 128, 129, 768, 1001, 1024, 1025, 4096, 17000, 32768])
@pytest.mark.parametrize("dtype", [BF, H, F])
def test_rows_exact(K, dtype):
    import kernels
    x = rows_of((13, K), dtype, K)
    x[1] = 0
    x[2] = torch.finfo(dtype).max
    if dtype != H:
        x[3] = 1e-37
        x[4] = x[4].float() * 1e-30
    x[5, K // 2], x[6, K - 1] = math.inf, math.nan
    codes, scale = orc.int8_rows(x)
    got = kernels.quantize_int8(x.cuda())
    assert got.codes.shape == x.shape and got.scale.shape == (13,) and got.dtype == dtype
    assert torch.equal(got.codes.cpu().double(), codes)
    assert torch.equal(torch.nan_to_num(got.scale.cpu(), nan=-1.0), torch.nan_to_num(scale, nan=-1.0))


# tokens around the tiles' widths (16 to 256), one or two short of and over them; outputs around a tile's 128
# channels and odd ones; K around a step's 128 and where it is split between blocks; outputs whose rows do not start on
# 16 bytes
SHAPES = [(1, 768, 32000), (1, 1, 1), (2, 16, 8), (15, 128, 128), (16, 4096, 4096), (17, 129, 130), (31, 1001, 257), (32, 256, 127),
          (33, 33, 129), (63, 768, 2304), (64, 16384, 64), (65, 640, 1000), (127, 2048, 384), (128, 100, 129), (129, 768, 513),
          (200, 8192, 100), (255, 768, 2304), (257, 384, 4097), (300, 1024, 16), (700, 512, 1280), (2931, 768, 2304), (5000, 64, 640),
          (3, 32768, 40),
          # two blocks a tile: a last tile with few tokens, or none, for its second block, and channels for one of them
          (2690, 1024, 4360), (2600, 1056, 4104), (5120, 1100, 2048),
          # fewer tokens than a tile and many channels; a weight larger than L2 keeps, tokens in two groups of tiles
          (100, 256, 19000), (2300, 32768, 1544),
          # a decoding step's kernel: clusters of 8, 4, 2 and 1 blocks a tile, and K on either side of its widest
          (16, 4096, 2048), (9, 1024, 2049), (16, 4095, 4096), (3, 2000, 8190), (7, 256, 20000), (16, 130, 64), (16, 4097, 4096)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F])
def test_product(M, K, N, dtype):
    import kernels
    x = rows_of((M, K), dtype, M + K)
    wc, wsc, w = weight(N, K, N)
    bias = params((N,), dtype, 5)[1]
    want, tol = orc.int8_product(*orc.int8_rows(x), wc, wsc, bias, dtype)
    got = kernels.int8_linear(x.cuda(), w, bias.cuda())
    assert got.dtype == dtype
    close(got, want, tol, "from x")
    # the same from rows made before, and again: the same bits
    rows = kernels.quantize_int8(x.cuda())
    assert torch.equal(kernels.int8_linear(rows, w, bias.cuda()), got)
    for _ in range(3):
        assert torch.equal(kernels.int8_linear(x.cuda(), w, bias.cuda()), got)


@pytest.mark.parametrize("dtype,bias_dtype", [(H, None), (H, H), (H, F), (BF, None), (BF, F), (F, F)])
@pytest.mark.parametrize("M", [5, 140])
def test_types_and_bias(M, dtype, bias_dtype):
    import kernels
    x = rows_of((M, 300), dtype, 1)
    wc, wsc, w = weight(77, 300, 2)
    bias = None if bias_dtype is None else params((77,), bias_dtype, 3)[1]
    want, tol = orc.int8_product(*orc.int8_rows(x), wc, wsc, bias, dtype)
    close(kernels.int8_linear(x.cuda(), w, None if bias is None else bias.cuda()), want, tol, "out")


@pytest.mark.parametrize("D", [8, 100, 768, 1001, 2048, 20000])
@pytest.mark.parametrize("dtype,wdtype", [(BF, F), (H, H), (F, F)])
def test_norm_rows(D, dtype, wdtype):
    """layer_norm_int8: each value within half a unit of the 64-bit norm's, beside that norm's own bound; and
    with the product after it, as they are used together."""
    import kernels
    x, (w, b) = rows_of((21, D), dtype, D), params((D,), wdtype, D + 1)
    y, tol, _ = orc.layer_norm(x, w, b, 1e-5, F)
    q = kernels.layer_norm_int8(*cuda(x, w, b))
    unit = q.scale.cpu().double()[:, None]
    got = q.codes.cpu().double() * unit
    # half a unit, the rounding of v * (127 / a), and a's own error on the unit
    assert ((got - y).abs() <= unit * (0.5 + 127 * 3 * orc.U) + tol * (1 + 1e-3) + tol.amax(-1, keepdim=True)).all()
    assert (q.codes.cpu().abs().amax(-1) == 127).all()
    wc, wsc, wt = weight(130, D, 3)
    want, tl = orc.int8_product(q.codes.cpu(), q.scale.cpu(), wc, wsc, None, dtype)
    close(kernels.int8_linear(q, wt), want, tl, "product")


def test_norm_rows_groups():
    import kernels
    x, (w, b) = rows_of((3, 5, 520), BF, 1), params((3, 520), F, 2)
    y = orc.layer_norm(x, w, b, 1e-5, F)[0]
    q = kernels.layer_norm_int8(*cuda(x, w, b))
    assert q.codes.shape == x.shape and q.scale.shape == (3, 5)
    assert ((q.dequantize().cpu().double() - y).abs() <= q.scale.cpu().double()[..., None] * 0.51).all()


def test_values():
    """Rows of zeros give the bias; a row with an infinity or NaN gives NaN in its own outputs alone; the
    largest sums (every code 127) are exact."""
    import kernels
    wc, wsc, w = weight(200, 256, 1)
    bias = torch.randn(200)
    x = torch.randn(20, 256)
    x[3] = 0
    x[4, 9], x[17, 255] = math.inf, math.nan
    got = kernels.int8_linear(x.cuda(), w, bias.cuda()).cpu()
    assert torch.equal(got[3], bias)
    assert torch.isnan(got[[4, 17]]).all() and torch.isfinite(got[[i for i in range(20) if i not in (4, 17)]]).all()
    ones = kernels.Int8Rows(torch.full((40, 32768), 127, dtype=torch.int8, device="cuda"), torch.ones(40, device="cuda"), F)
    assert torch.equal(kernels.int8_linear(ones, ones), torch.full((40, 40), 127.0 * 127 * 32768, device="cuda"))


def test_layouts():
    """Strided x, leading axes, codes whose rows do not start on 16 bytes, empty inputs, one axis."""
    import kernels
    wc, wsc, w = weight(50, 96, 1)
    base = rows_of((40, 131), BF, 2)
    for view in (lambda t: t[:, :96], lambda t: t[:, 3:99], lambda t: t[::3, :96], lambda t: t[:, :96].unflatten(0, (5, 8)).transpose(0, 1),
                 lambda t: t[7, :96], lambda t: t[:0, :96], lambda t: t[2:3, :96].expand(30, 96)):
        x = view(base)
        want, tol = orc.int8_product(*orc.int8_rows(x), wc, wsc, None, BF)
        close(kernels.int8_linear(view(base.cuda()), w), want, tol, "x")
        q = kernels.quantize_int8(view(base.cuda()))
        close(kernels.int8_linear(q, w), want, tol, "rows")
        loose = kernels.Int8Rows(torch.nn.functional.pad(q.codes, (1, 2))[..., 1:-2], q.scale, q.dtype)
        close(kernels.int8_linear(loose, kernels.Int8Rows(w.codes.t().contiguous().t(), w.scale)), want, tol, "loose codes")
    none = kernels.Int8Rows(torch.empty(0, 96, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"))
    assert kernels.int8_linear(base[:, :96].cuda(), none).shape == (40, 0)


def test_bytes_beyond_a_row_are_not_read():
    """K is not a multiple of 16: what lies in the rows' padding has no effect."""
    import kernels
    x = rows_of((9, 77), F, 1)
    wc, wsc, w = weight(33, 77, 2)
    want, tol = orc.int8_product(*orc.int8_rows(x), wc, wsc, None, F)
    q = kernels.quantize_int8(x.cuda())
    for t in (q, w):
        t.codes.as_strided((t.codes.shape[0], 80), (80, 1))[:, 77:] = 99
    close(kernels.int8_linear(q, w), want, tol, "out")


def test_streams_graphs_and_together():
    """Two streams at once, and two captured graphs replayed in turn, on few tokens (K split between blocks)
    and many."""
    import kernels
    wc, wsc, w = weight(1000, 2048, 1)
    xs = [rows_of((m, 2048), BF, m).cuda() for m in (3, 300)]
    want = [kernels.int8_linear(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kernels.int8_linear(xs[i], w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            y = kernels.int8_linear(x, w)
        graphs.append((g, y))
    fresh = [rows_of((x.shape[0], 2048), BF, 7).cuda() for x in xs]
    for x, f in zip(xs, fresh):
        x.copy_(f)
    for i in (1, 0, 1, 0):
        graphs[i][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[i][1], kernels.int8_linear(fresh[i], w))


def test_error_word():
    """check_timeout reads the kernel's error word back: no wait gave up."""
    import flb_native as nat
    import kernels
    for M in (1, 64, 600):
        x = rows_of((M, 640), BF, 1).cuda()
        _, _, w = weight(300, 640, 2)
        out = torch.empty(M, 300, dtype=BF, device="cuda")
        n = nat.lib.flb_int8_linear_workspace_bytes(M, 300, 640, 0)
        ws = nat.workspace(n, x.device)
        nat.check(nat.lib.flb_int8_linear(x.data_ptr(), 640, None, 0, None, w.codes.data_ptr(), 640, w.scale.data_ptr(), None, 0,
                                          out.data_ptr(), M, 300, 640, nat.BF16, ws.data_ptr(), n, 1, nat.stream_of(x)), "int8")
        assert torch.equal(out, kernels.int8_linear(x, w))


def test_refusals():
    import kernels
    x = torch.zeros(4, 32, device="cuda")
    w = kernels.quantize_int8(torch.ones(8, 32, device="cuda"))
    for bad in (kernels.Int8Rows(w.codes[:, :16], w.scale), kernels.Int8Rows(w.codes, w.scale[:4]), kernels.Int8Rows(w.codes[0], w.scale[0]),
                kernels.Int8Rows(w.codes[None], w.scale[None])):
        with pytest.raises(ValueError):
            kernels.int8_linear(x, bad)
    for bad in (kernels.Int8Rows(w.codes.short(), w.scale), kernels.Int8Rows(w.codes, w.scale.double())):
        with pytest.raises(TypeError):
            kernels.int8_linear(x, bad)
    with pytest.raises(ValueError):
        kernels.int8_linear(x, w, torch.zeros(7, device="cuda"))
    with pytest.raises(TypeError):
        kernels.int8_linear(x, w, torch.zeros(8, device="cuda", dtype=BF))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kernels.int8_linear(x, kernels.Int8Rows(w.codes.cpu(), w.scale.cpu()))
    with pytest.raises(TypeError):
        kernels.quantize_int8(x.double())
    with pytest.raises(ValueError):
        kernels.quantize_int8(x[:, :0])
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        kernels.quantize_int8(torch.zeros(1, 32769, device="cuda"))


def test_module_and_gradients():
    import kernels
    torch.manual_seed(0)
    lin = torch.nn.Linear(768, 320, device="cuda", dtype=BF)
    q = kernels.Int8Linear.from_linear(lin)
    x = torch.randn(4, 7, 768, device="cuda", dtype=BF)
    got, want = q(x), lin(x)
    assert got.shape == want.shape and got.dtype == want.dtype
    assert (got - want).float().norm() <= 0.02 * want.float().norm()  # two roundings of 1/127 of the rows' largest, averaged over 768
    assert torch.equal(q(x.float()), kernels.int8_linear(x.float(), kernels.Int8Rows(q.codes, q.scale), q.bias.float()))
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        kernels.int8_linear(x, kernels.Int8Rows(q.codes, q.scale))
    with pytest.raises(RuntimeError, match="no gradient"):
        kernels.layer_norm_int8(x)
    with torch.no_grad():
        kernels.int8_linear(x, kernels.Int8Rows(q.codes, q.scale))
