"""LayerNorm, the 8-bit kept form and the sigmoid gate on a B200, against 64-bit definitions with derived
bounds (oracle/rows.py)."""
import math

import pytest
import torch

from oracle import rows as orc

pytestmark = pytest.mark.gpu

BF, H, F = torch.bfloat16, torch.float16, torch.float32


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def close(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    over = (got - want).abs() - tol
    over = torch.where(torch.isnan(want) & torch.isnan(got), torch.full_like(over, -1.0), over)
    assert not torch.isnan(over).any() and (over.numel() == 0 or over.max() <= 0), \
        f"{what}: {over.max():.3g} over its bound at {int(over.argmax())}"


def rows_of(shape, dtype, seed, spread=1.0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * spread
    x = x * (1 + 15 * (torch.rand(shape[-1], generator=g) < 0.02)) + offset
    return x.to(dtype)


def params(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(*shape, generator=g)).to(dtype), (0.2 * torch.randn(*shape, generator=g)).to(dtype)


# widths around a lane's 8, a warp's 256, a warp's row of 1024, a block's row, the widest; odd ones unaligned
WIDTHS = [1, 2, 7, 8, 31, 33, 127, 128, 129, 255, 256, 264, 513, 768, 1000, 1001, 1024, 1025, 1032, 2048, 4097, 8192, 8200, 16384]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,wdtype", [(BF, F), (BF, BF), (H, H), (H, F), (F, F)])
def test_norm_forward_backward(D, dtype, wdtype):
    import kernels
    R = 37 if D < 4000 else 9
    x, (w, b) = rows_of((R, D), dtype, D), params((D,), wdtype, D + 1)
    dy = rows_of((R, D), dtype, D + 2)
    y, tol, back = orc.layer_norm(x, w, b, 1e-5, dtype)
    xs, ws, bs, dys = cuda(x, w, b, dy)
    close(kernels.layer_norm(xs, ws, bs), y, tol, "inference")
    for t in (xs, ws, bs):
        t.requires_grad_(True)
    got = kernels.layer_norm(xs, ws, bs)
    close(got, y, tol, "y")
    got.backward(dys)
    want = orc.layer_norm_backward(*back, w, dy, dtype, wdtype)
    for t, (v, tl), name in zip((xs, ws, bs), want, ("dx", "dw", "db")):
        assert t.grad.dtype == t.dtype
        close(t.grad, v, tl, name)


@pytest.mark.parametrize("D", [1, 17, 128, 129, 768, 1001, 1024, 1280, 4096, 8200])
@pytest.mark.parametrize("dtype,wdtype", [(BF, F), (H, H), (F, F)])
def test_norm_kept(D, dtype, wdtype):
    import kernels
    R = 41
    x, (w, b) = rows_of((R, D), dtype, D), params((D,), wdtype, D + 1)
    dy = rows_of((R, D), dtype, D + 2)
    y, tol, back = orc.layer_norm(x, w, b, 1e-5, dtype)
    xs, ws, bs, dys = (t.requires_grad_(True) for t in cuda(x, w, b, dy))
    got = kernels.layer_norm(xs, ws, bs, keep8=True)
    close(got, y, tol, "y")
    grads = torch.autograd.grad(got, (xs, ws, bs), dys.detach())
    want = orc.layer_norm_backward(*back, w, dy, dtype, wdtype, keep8=True)
    for g, (v, tl), name in zip(grads, want, ("dx", "dw", "db")):
        close(g, v, tl, name)
    # and what 8 bits cost: rounding puts every h off by half its unit at most, so dw = sum dy h is off by
    # sum |dy| unit / 2 at most, beside the bound of the kept form's own gradient (loud channels among 128
    # share their unit with the others: a fixed share of the gradient's norm does not follow)
    unit = orc.kept(back[0])[1]
    full = orc.layer_norm_backward(*back, w, dy, dtype, wdtype)[1][0]
    close(grads[1], full, (dy.double().abs() * unit / 2).sum(0) + want[1][1], "dw against the one from x")


@pytest.mark.parametrize("shape", [(1, 1), (1, 5), (4, 1), (3, 600), (7, 200), (2, 5000)])
@pytest.mark.parametrize("D", [24, 768, 1001, 2056])
@pytest.mark.parametrize("keep8", [False, True])
def test_norm_groups(shape, D, keep8):
    """A weight for each of G groups; few rows (one block a group) and many (sums through the workspace)."""
    import kernels
    if D > 1000 and shape[1] > 1000:
        shape = (2, 300)
    x, (w, b) = rows_of((*shape, D), BF, 3), params((shape[0], D), F, 4)
    dy = rows_of((*shape, D), BF, 5)
    y, tol, back = orc.layer_norm(x, w, b, 1e-5, BF)
    xs, ws, bs, dys = cuda(x, w, b, dy)
    for t in (xs, ws, bs):
        t.requires_grad_(True)
    got = kernels.layer_norm(xs, ws, bs, keep8=keep8)
    close(got, y, tol, "y")
    grads = torch.autograd.grad(got, (xs, ws, bs), dys)
    want = orc.layer_norm_backward(*back, w, dy, BF, F, keep8=keep8, groups=tuple(w.shape))
    for g, (v, tl), name in zip(grads, want, ("dx", "dw", "db")):
        close(g, v, tl, name)


def test_norm_deterministic_and_empty():
    import kernels
    x, w, b, dy = cuda(rows_of((5000, 768), BF, 1), *params((768,), F, 2), rows_of((5000, 768), BF, 3))
    w.requires_grad_(True), b.requires_grad_(True)
    first = torch.autograd.grad(kernels.layer_norm(x, w, b), (w, b), dy)
    for _ in range(3):
        again = torch.autograd.grad(kernels.layer_norm(x, w, b), (w, b), dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
    for shape in ((0, 768), (3, 0, 768)):
        e = torch.empty(shape, device="cuda", dtype=BF, requires_grad=True)
        y = kernels.layer_norm(e, w, b, keep8=True)
        gx, gw, gb = torch.autograd.grad(y, (e, w, b), torch.empty_like(y))
        assert y.shape == e.shape == gx.shape and not gw.any() and not gb.any()


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_norm_without_parameters(which):
    import kernels
    x, (w, b), dy = rows_of((50, 520), H, 1), params((520,), H, 2), rows_of((50, 520), H, 3)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    y, tol, back = orc.layer_norm(x, w, b, 1e-3, H)
    xs, ws, bs, dys = cuda(x, w, b, dy)
    leaves = [t.requires_grad_(True) for t in (xs, ws, bs) if t is not None]
    got = kernels.layer_norm(xs, ws, bs, eps=1e-3)
    close(got, y, tol, "y")
    grads = torch.autograd.grad(got, leaves, dys)
    dx, dw, db = orc.layer_norm_backward(*back, w, dy, H, H)
    want = [dx] + ([dw] if w is not None else []) + ([db] if b is not None else [])
    for g, (v, tl) in zip(grads, want):
        close(g, v, tl, which)


def test_norm_strides_and_offsets():
    """Row pitches, transposed and expanded inputs, storages that start off 16 bytes, expanded gradients."""
    import kernels
    w, b = params((96,), F, 1)
    base = rows_of((40, 131), BF, 2)
    wc, bc = cuda(w, b)
    views = {"pitch": lambda t: t[:, :96], "offset": lambda t: t[:, 3:99], "aligned offset": lambda t: t[:, 8:104],
             "every other row": lambda t: t[::2, :96], "three axes": lambda t: t[:, :96].unflatten(0, (5, 8)),
             "transposed": lambda t: t[:, :96].unflatten(0, (5, 8)).transpose(0, 1), "one row many times": lambda t: t[3:4, :96].expand(9, 96),
             "columns apart": lambda t: t.t()[:40, :96] if t.shape[0] >= 96 else t[:, ::1][:, :96]}
    for name, view in views.items():
        x = view(base)
        y, tol, back = orc.layer_norm(x, w, b, 1e-5, BF)
        xs = view(base.cuda()).detach().requires_grad_(True)
        got = kernels.layer_norm(xs, wc, bc)
        close(got, y, tol, name)
        (gx,) = torch.autograd.grad(got.sum(), xs)  # an expanded gradient
        (dx, tl), _, _ = orc.layer_norm_backward(*back, w, torch.ones_like(x), BF, F)
        close(gx, dx, tl, name + " dx")
    square = rows_of((96, 96), F, 6)
    got = kernels.layer_norm(square.cuda().t(), wc, bc)
    y, tol, _ = orc.layer_norm(square.t(), w, b, 1e-5, F)
    close(got, y, tol, "transposed matrix")


def test_norm_values():
    """Constant rows, rows far from zero, tiny and huge rows, infinities and NaN stay in their own row."""
    import kernels
    D = 640
    x = torch.randn(8, D, generator=torch.Generator().manual_seed(0))
    x[0] = 3.0
    x[1] = x[1] * 1e-3 + 1000.0
    x[2] *= 1e-12
    x[3] *= 1e15
    x[4] = 0
    x[5, 17], x[6, 639] = math.inf, math.nan
    y, tol, _ = orc.layer_norm(x, None, None, 1e-5, F)
    for keep8 in (False, True):
        xs = x.cuda().requires_grad_(True)
        got = kernels.layer_norm(xs, keep8=keep8)
        fine = [0, 1, 2, 3, 4, 7]
        close(got[fine], y[fine], tol[fine], "y")
        assert torch.isnan(got[5]).all() and torch.isnan(got[6]).all()
        (gx,) = torch.autograd.grad(got, xs, torch.randn(8, D, device="cuda"))
        assert torch.isfinite(gx[fine]).all() and torch.isnan(gx[5]).all() and torch.isnan(gx[6]).all()


def test_norm_against_differences():
    """The gradient against central differences of the 64-bit forward."""
    import kernels
    x, (w, b), dy = rows_of((3, 20), F, 1), params((20,), F, 2), rows_of((3, 20), F, 3)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(kernels.layer_norm(*leaves), leaves, dy.cuda())

    def loss(*v):
        return (orc.layer_norm(v[0], v[1], v[2], 1e-5, F)[0] * dy.double()).sum()

    vals, step = [t.double() for t in (x, w, b)], 1e-5
    for k, g in enumerate(grads):
        for i in range(0, vals[k].numel(), 7):
            up, down = [v.clone() for v in vals], [v.clone() for v in vals]
            up[k].view(-1)[i] += step
            down[k].view(-1)[i] -= step
            # differences are good to step^2 and 1e-16 / step of the loss (a few tens)
            assert abs((loss(*up) - loss(*down)).item() / (2 * step) - g.view(-1)[i].item()) < 1e-4 * (1 + abs(g.view(-1)[i].item()))


def test_norm_vmap_and_vjp():
    import kernels
    G, R, D = 4, 6, 96
    x, (w, b), dy = rows_of((G, R, D), F, 1), params((G, D), F, 2), rows_of((G, R, D), F, 3)
    xs, ws, bs, dys = cuda(x, w, b, dy)
    y, tol, back = orc.layer_norm(x, w, b, 1e-5, F)
    for keep8 in (False, True):
        f = torch.vmap(lambda p, q, r: kernels.layer_norm(p, q, r, keep8=keep8))
        close(f(xs, ws, bs), y, tol, "vmap")
        out, pull = torch.func.vjp(f, xs, ws, bs)
        close(out, y, tol, "vjp")
        want = orc.layer_norm_backward(*back, w, dy, F, F, keep8=keep8, groups=(G, D))
        for g, (v, tl) in zip(pull(dys), want):
            close(g, v, tl, "vjp")
    # a mapped x with one weight, a mapped weight with one x, a mapped axis that is not the first
    y1, tol1, _ = orc.layer_norm(x, w[0], b[0], 1e-5, F)
    close(torch.vmap(lambda p: kernels.layer_norm(p, ws[0], bs[0]))(xs), y1, tol1, "one weight")
    close(torch.vmap(lambda p: kernels.layer_norm(p, ws[0], bs[0]), in_dims=1, out_dims=1)(xs), y1, tol1, "axis 1")
    y2, tol2, _ = orc.layer_norm(x[:1].expand(G, R, D), w, b, 1e-5, F)
    close(torch.vmap(lambda q, r: kernels.layer_norm(xs[0], q, r))(ws, bs), y2, tol2, "one x")
    # groups inside a vmap, and a vmap inside a vmap
    big, wb = torch.stack([x, x + 1]), torch.stack([w, w + 1])
    y3, tol3, _ = orc.layer_norm(big.reshape(2 * G, R, D), wb.reshape(2 * G, D), None, 1e-5, F)
    close(torch.vmap(lambda p, q: kernels.layer_norm(p, q))(big.cuda(), wb.cuda()).reshape(2 * G, R, D), y3, tol3, "groups")
    close(torch.vmap(torch.vmap(lambda p, q: kernels.layer_norm(p, q)))(big.cuda(), wb.cuda()).reshape(2 * G, R, D), y3, tol3, "twice")


def special(dtype):
    """Blocks that test the kept form's rule: borders of the unit, ties, zeros, subnormals, extremes."""
    fi = torch.finfo(dtype)
    rows = [torch.zeros(128), torch.full((128,), fi.max), torch.full((128,), -fi.max), torch.full((128,), fi.tiny),
            torch.full((128,), fi.smallest_normal * fi.eps), torch.linspace(-127.5, 127.5, 128), torch.arange(128) - 63.5,
            torch.arange(128) * 0.5, torch.full((128,), 127.0), torch.full((128,), 127.5), torch.full((128,), 126.99),
            torch.full((128,), 63.75), torch.full((128,), 0.99609375), torch.full((128,), 0.9960), torch.full((128,), 1e-3)]
    inf, nan = torch.ones(128), torch.ones(128)
    inf[5], nan[127] = math.inf, math.nan
    return torch.stack([r.to(dtype) for r in rows + [inf, nan]])


@pytest.mark.parametrize("D", [1, 5, 17, 127, 128, 129, 256, 300, 768, 1001, 2304, 40000])
@pytest.mark.parametrize("dtype", [BF, H, F])
def test_pack_exact(D, dtype):
    import kernels
    x = torch.cat([rows_of((19, D), dtype, D), special(dtype).repeat(1, -(-D // 128))[:, :D]])
    want = orc.kept(x)[0]
    lim = torch.finfo(dtype).max
    want = torch.where(torch.isnan(want), want, want.clamp(-lim, lim)).to(dtype)
    p = kernels.pack8(x.cuda())
    assert p.codes.shape[1] % 16 == 0 and p.codes.dtype == torch.int8
    got = kernels.unpack8(p).cpu()
    assert got.dtype == dtype and torch.equal(torch.nan_to_num(got, nan=1.5), torch.nan_to_num(want, nan=1.5))
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    wide = kernels.unpack8(p, torch.float32).cpu()  # exact in 32 bits
    assert torch.equal(torch.nan_to_num(wide.double(), nan=1.5), torch.nan_to_num(orc.kept(x)[0], nan=1.5))


def test_pack_shapes():
    import kernels
    for shape in ((0,), (5,), (0, 7), (3, 0), (2, 3, 4, 129)):
        x = torch.randn(shape, device="cuda")
        assert kernels.unpack8(kernels.pack8(x)).shape == x.shape
    x = torch.randn(40, 300, device="cuda")[:, 1:290].t()
    assert torch.equal(kernels.unpack8(kernels.pack8(x)), kernels.unpack8(kernels.pack8(x.contiguous())))


@pytest.mark.parametrize("shape", [(1, 1), (3, 17), (96, 768), (5, 7, 129), (33, 1001), (700, 2048)])
@pytest.mark.parametrize("dtype", [BF, H, F])
@pytest.mark.parametrize("keep8", [False, True])
def test_gate(shape, dtype, keep8):
    import kernels
    x, z, dy = (rows_of(shape, dtype, s) for s in (1, 2, 3))
    xs, zs, dys = cuda(x, z, dy)
    y, tol = orc.gate(x, z, dtype)
    close(kernels.sigmoid_gate(xs, zs), y, tol, "inference")
    xs.requires_grad_(True), zs.requires_grad_(True)
    got = kernels.sigmoid_gate(xs, zs, keep8=keep8)
    close(got, y, tol, "y")
    for g, (v, tl), name in zip(torch.autograd.grad(got, (xs, zs), dys), orc.gate_backward(x, z, dy, dtype, keep8), ("dx", "dz")):
        close(g, v, tl, name)


def test_gate_values():
    """Large |z|: neither side of the gate overflows or is lost; a NaN reaches only its own element or block."""
    import kernels
    z = torch.tensor([-200.0, -90.0, -30.0, -1.0, 0.0, 1.0, 16.0, 30.0, 90.0, 200.0])
    x = torch.full_like(z, 2.0)
    xs, zs = x.cuda().requires_grad_(True), z.cuda().requires_grad_(True)
    y = kernels.sigmoid_gate(xs, zs)
    dx, dz = torch.autograd.grad(y, (xs, zs), torch.ones_like(y))
    (wx, tx), (wz, tz) = orc.gate_backward(x, z, torch.ones_like(x), F)
    close(dx, wx, tx + 1e-38, "dx"), close(dz, wz, tz + 1e-38, "dz")
    x = torch.randn(2, 300)
    x[0, 3], x[1, 290] = math.nan, math.inf
    xs, zs = x.cuda().requires_grad_(True), torch.randn(2, 300, device="cuda", requires_grad=True)
    y = kernels.sigmoid_gate(xs, zs, keep8=True)
    assert torch.isnan(y).sum() == 1 and torch.isinf(y).sum() == 1
    dx, dz = torch.autograd.grad(y, (xs, zs), torch.ones_like(y))
    assert torch.isfinite(dx).all() and torch.isnan(dz).sum() == 128 + 44


def test_gate_vmap():
    import kernels
    x, z, dy = (rows_of((3, 4, 200), F, s) for s in (1, 2, 3))
    xs, zs, dys = cuda(x, z, dy)
    y, tol = orc.gate(x, z, F)
    for keep8 in (False, True):
        out, pull = torch.func.vjp(torch.vmap(lambda p, q: kernels.sigmoid_gate(p, q, keep8=keep8)), xs, zs)
        close(out, y, tol, "vmap")
        for g, (v, tl) in zip(pull(dys), orc.gate_backward(x, z, dy, F, keep8)):
            close(g, v, tl, "vjp")


def test_streams_graphs_and_memory():
    """Another stream, and forward and backward captured into a graph and replayed on new inputs, also with
    two graphs alive; with keep8 the forward keeps about a byte an element."""
    import kernels
    x, w, b, z = cuda(rows_of((300, 768), BF, 1), *params((768,), F, 2), rows_of((300, 768), BF, 4))
    dy = rows_of((300, 768), BF, 5).cuda()
    leaves = [t.requires_grad_(True) for t in (x, w, b, z)]

    def step(keep8):
        y = kernels.sigmoid_gate(kernels.layer_norm(x, w, b, keep8=keep8), z, keep8=keep8)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = {k: [t.clone() for t in step(k)] for k in (False, True)}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = {}
    with torch.cuda.stream(s):
        for k in (False, True):
            got = step(k)
            s.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want[k]))
            del got
    torch.cuda.synchronize()
    for k in (False, True):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = step(k)
        graphs[k] = (g, out)
    with torch.no_grad():
        x.copy_(rows_of((300, 768), BF, 9))
    fresh = {k: [t.clone() for t in step(k)] for k in (False, True)}
    for k in (True, False, True):
        g, out = graphs[k]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, fresh[k]))
    big = torch.randn(4096, 1024, device="cuda", dtype=BF, requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = kernels.layer_norm(big * 1, keep8=True)  # the product itself is not kept
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert kept <= big.numel() * (1 + 1 / 128) + 4096 * 4 + 4096, kept


@pytest.mark.parametrize("offset", [30.0, 3000.0])
def test_norm_far_from_zero(offset):
    """Rows whose offset is many times their spread: the bounds grow with the offset, as the mean's rounding does."""
    import kernels
    for D in (200, 1001, 4096):
        x, (w, b), dy = rows_of((33, D), F, 1, offset=offset), params((D,), F, 2), rows_of((33, D), F, 3)
        y, tol, back = orc.layer_norm(x, w, b, 1e-5, F)
        xs, ws, bs, dys = cuda(x, w, b, dy)
        for t in (xs, ws, bs):
            t.requires_grad_(True)
        got = kernels.layer_norm(xs, ws, bs)
        close(got, y, tol, "y")
        for g, (v, tl), name in zip(torch.autograd.grad(got, (xs, ws, bs), dys), orc.layer_norm_backward(*back, w, dy, F, F), ("dx", "dw", "db")):
            close(g, v, tl, name)


def test_norm_widest():
    import kernels
    x, (w, b) = rows_of((5, 32768), F, 1), params((32768,), F, 2)
    y, tol, _ = orc.layer_norm(x, w, b, 1e-5, F)
    close(kernels.layer_norm(*cuda(x, w, b)), y, tol, "y")
    with pytest.raises(RuntimeError, match="wider than 16384"):
        kernels.layer_norm(torch.zeros(2, 16385, device="cuda", requires_grad=True))
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        kernels.layer_norm(torch.zeros(2, 32769, device="cuda"))


def test_frozen_leaves_and_in_place():
    """Gradients for the input alone, the parameters alone, one of them; an input changed after the forward is
    noticed where the backward reads it, and allowed where it does not; a second derivative is refused."""
    import kernels
    x, (w, b), dy = rows_of((64, 256), F, 1), params((256,), F, 2), rows_of((64, 256), F, 3)
    _, _, back = orc.layer_norm(x, w, b, 1e-5, F)
    want = orc.layer_norm_backward(*back, w, dy, F, F)
    for wanted in ((0,), (1,), (2,), (1, 2), (0, 2)):
        ts = cuda(x, w, b)
        for i in wanted:
            ts[i].requires_grad_(True)
        grads = torch.autograd.grad(kernels.layer_norm(*ts), [ts[i] for i in wanted], dy.cuda())
        for g, i in zip(grads, wanted):
            close(g, *want[i], f"leaf {i}")
    for keep8 in (False, True):
        leaf = x.cuda().requires_grad_(True)
        mid = leaf * 1
        y = kernels.layer_norm(mid, keep8=keep8)
        mid.zero_()
        if keep8:
            y.backward(dy.cuda())
        else:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward(dy.cuda())
        xs, zs = x.cuda().requires_grad_(True), x.cuda().requires_grad_(True)
        for out in (kernels.layer_norm(xs, keep8=keep8), kernels.sigmoid_gate(xs, zs, keep8=keep8)):
            (g,) = torch.autograd.grad(out.square().sum(), xs, create_graph=True)
            with pytest.raises(RuntimeError, match="differentiable once"):
                g.sum().backward()


def test_refusals():
    import kernels
    x = torch.zeros(4, 8, device="cuda")
    for bad in (torch.ones(9, device="cuda"), torch.ones(3, 8, device="cuda"), torch.ones(4, 1, 8, device="cuda"), torch.tensor(1.0, device="cuda")):
        with pytest.raises(ValueError):
            kernels.layer_norm(x, bad)
    with pytest.raises(ValueError):
        kernels.layer_norm(x, torch.ones(8, device="cuda"), torch.ones(4, 8, device="cuda"))
    with pytest.raises(ValueError):
        kernels.layer_norm(x[:, :0])
    with pytest.raises(ValueError):
        kernels.layer_norm(torch.tensor(1.0, device="cuda"))
    with pytest.raises(TypeError):
        kernels.layer_norm(x, torch.ones(8, device="cuda", dtype=BF))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kernels.layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError):
        kernels.sigmoid_gate(x, x[:1])
    with pytest.raises(TypeError):
        kernels.sigmoid_gate(x, x.half())
    with pytest.raises(ValueError):
        kernels.pack8(torch.tensor(1.0, device="cuda"))
    # transforms that have no rule
    q = kernels.quantize_int8(x)
    for call in (lambda t: kernels.pack8(t).codes, lambda t: kernels.quantize_int8(t).codes, lambda t: kernels.layer_norm_int8(t).codes,
                 lambda t: kernels.int8_linear(t, q)):
        with pytest.raises(RuntimeError, match="torch.func transforms"):
            torch.vmap(call)(x)
    w = torch.ones(8, device="cuda")
    for f in (lambda t: kernels.layer_norm(t, w).sum(), lambda t: kernels.sigmoid_gate(t, t).sum()):
        with pytest.raises(RuntimeError, match="vmap over this operator's backward"):
            torch.vmap(torch.func.grad(f))(x)


def test_large_offsets():
    """Rows beyond 2^31 elements."""
    import kernels
    R, D = 70000, 32768
    x = torch.empty((R, D), dtype=BF, device="cuda")
    x[-3:] = torch.randn(3, D, device="cuda")
    tail = x[-3:].cpu()
    got = kernels.layer_norm(x)[-3:].clone()
    y, tol, _ = orc.layer_norm(tail, None, None, 1e-5, BF)
    close(got, y, tol, "y")
    p = kernels.pack8(x)
    del x
    last = kernels.Packed8(p.codes[-3:], p.exps[-3:], torch.Size((3, D)), BF)
    assert torch.equal(kernels.unpack8(last).cpu().double(), orc.kept(tail)[0])
