"""AdamW's step on a B200, against its formula in 64 bits; moments in 8 bits exactly."""
import copy
import math

import pytest
import torch

from oracle import head as orc

pytestmark = pytest.mark.gpu

BF, H, F = torch.bfloat16, torch.float16, torch.float32
SIZES = [(1,), (3,), (127,), (128,), (129,), (5, 31), (4095,), (4096,), (4097,), (33, 257), (0,), (100003,)]


def make(shapes, dtype, seed, grad=0.01):
    g = torch.Generator().manual_seed(seed)
    params = [(0.1 * torch.randn(s, generator=g)).to(dtype).cuda().requires_grad_(True) for s in shapes]
    return params, lambda: [(grad * torch.randn(p.shape, generator=g)).to(dtype) for p in params]


def before(opt, p, bits):
    """A parameter, its moments' values and steps taken, on the CPU."""
    s, n = opt.state.get(p, {}), p.numel()
    if not s:
        return p.detach().cpu().clone(), torch.zeros(p.shape), torch.zeros(p.shape), 0
    if bits == 8:
        m = orc.moment_values(s["exp_avg"], s["exp_avg_exps"], 14, False, n).float().view(p.shape)
        v = orc.moment_values(s["exp_avg_sq"], s["exp_avg_sq_exps"], 30, True, n).float().view(p.shape)
    else:
        m, v = s["exp_avg"].cpu().clone(), s["exp_avg_sq"].cpu().clone()
    return p.detach().cpu().clone(), m, v, int(s["step"])


def check(opt, p, was, g, bits, seed=0, lr=None):
    group = next(x for x in opt.param_groups if any(p is q for q in x["params"]))
    old, m, v, t = was
    s, t = opt.state[p], t + 1
    assert int(s["step"]) == t
    lr = float(group["lr"]) if lr is None else lr
    want, m64, v64, tol_p, tol_m, tol_v = orc.adamw(old, g, m, v, t, lr, group["betas"], group["eps"], group["weight_decay"])
    got = p.detach().cpu().double()
    # p's own rounding: half a step of its type, and of the smallest numbers
    tol_p = tol_p + torch.finfo(p.dtype).eps / 2 * (want.abs() + tol_p) + torch.finfo(p.dtype).smallest_normal * torch.finfo(p.dtype).eps
    assert ((got - want).abs() <= tol_p).all(), ((got - want).abs() / tol_p).max()
    if bits == 32:
        assert ((s["exp_avg"].cpu().double() - m64).abs() <= tol_m + 2.0 ** -149).all()
        assert ((s["exp_avg_sq"].cpu().double() - v64).abs() <= tol_v + 2.0 ** -148).all()
    else:
        m32, v32 = orc.moments32(g, m, v, group["betas"])
        rm, rv = orc.noise(p.numel(), t, seed)
        for name, x, r, form in (("exp_avg", m32, rm, (14, False)), ("exp_avg_sq", v32, rv, (30, True))):
            codes, exps = orc.moment_codes(x, r, *form)
            assert torch.equal(s[name + "_exps"].cpu().long(), exps)
            fine = (exps != 255)[:, None]
            assert torch.equal(s[name].cpu().long() * fine, codes * fine)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F, BF, H])
def test_steps(dtype, bits):
    import kernels
    params, grads = make(SIZES, dtype, 1)
    opt = kernels.AdamW(params, lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1, state_bits=bits, seed=77)
    for _ in range(4):
        gs = grads()
        for p, g in zip(params, gs):
            p.grad = g.cuda()
        was = [before(opt, p, bits) for p in params]
        opt.step()
        for p, w, g in zip(params, was, gs):
            check(opt, p, w, g, bits, seed=77)
    for (m, v), p in zip(opt.moments(), params):
        _, wm, wv, _ = before(opt, p, bits)
        assert torch.equal(m.cpu(), wm) and torch.equal(v.cpu(), wv)


@pytest.mark.parametrize("bits", [32, 8])
def test_other_settings_and_missing_gradients(bits):
    import kernels
    params, grads = make([(300,), (40, 7), (1000,)], F, 2)
    opt = kernels.AdamW([{"params": params[:2], "lr": 0.1, "betas": (0.0, 0.0), "eps": 1e-3}, {"params": params[2:], "weight_decay": 0.0}], state_bits=bits)
    for i in range(4):
        gs = grads()
        was = [before(opt, p, bits) for p in params]
        for j, (p, g) in enumerate(zip(params, gs)):
            p.grad = None if (i + j) % 3 == 0 else g.cuda()
        opt.step()
        for p, w, g in zip(params, was, gs):
            if p.grad is not None:
                check(opt, p, w, g, bits)
            else:
                assert torch.equal(p.detach().cpu(), w[0]) and (not opt.state.get(p) or int(opt.state[p]["step"]) == w[3])
    kernels.AdamW([torch.zeros(3, device="cuda")]).step()  # nothing to do


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F, BF])
def test_layouts(dtype, bits):
    """Parameters that do not start on 16 bytes, transposed ones, and gradients laid out in another way."""
    import kernels
    base = torch.randn(5000, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    kept = base.cpu().clone()
    params = [base[1:1000], base[1003:1300], base[2000:2000 + 33 * 40].view(33, 40).t(), base[4000:4001]]
    opt = kernels.AdamW(params, lr=1e-2, state_bits=bits)
    g = torch.Generator().manual_seed(4)
    for _ in range(3):
        was = [before(opt, p, bits) for p in params]
        gs = [(0.1 * torch.randn(p.shape, generator=g)).to(dtype) for p in params]
        for p, x in zip(params, gs):
            p.grad = x.cuda()
        opt.step()
        for p, w, x in zip(params, was, gs):
            if bits == 8 and not p.is_contiguous():
                # codes go by the parameter's memory
                p, x, w = p.t(), x.t().contiguous(), (w[0].t(), *(y.reshape(-1).view(p.t().shape) for y in w[1:3]), w[3])
                opt.state[p] = opt.state[params[2]]
                opt.param_groups[0]["params"].append(p)
                check(opt, p, w, x, bits)
                opt.param_groups[0]["params"].pop()
                del opt.state[p]
            else:
                check(opt, p, w, x, bits)
    untouched = torch.ones(5000, dtype=torch.bool)
    for lo, hi in ((1, 1000), (1003, 1300), (2000, 3320), (4000, 4001)):
        untouched[lo:hi] = False
    assert torch.equal(base.cpu()[untouched], kept[untouched])


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes(bits):
    import kernels
    params, grads = make([(1 + i % 300,) for i in range(1000)], F, 5)
    opt = kernels.AdamW(params, state_bits=bits)
    for _ in range(2):
        gs = grads()
        was = [before(opt, p, bits) for p in params]
        for p, g in zip(params, gs):
            p.grad = g.cuda()
        opt.step()
        for i in (0, 47, 48, 439, 440, 441, 879, 880, 999):
            check(opt, params[i], was[i], gs[i], bits)
    assert all(int(opt.state[p]["step"]) == 2 for p in params)


def test_extremes():
    """Infinities and NaN stay in their element (32 bits) or its block (8 bits); large and small gradients are exact codes."""
    import kernels
    for bits in (32, 8):
        p = torch.zeros(1280, device="cuda")
        opt = kernels.AdamW([p], state_bits=bits, eps=0.0 if bits == 32 else 1e-8)
        g = torch.randn(1280, generator=torch.Generator().manual_seed(6))
        g[5], g[200], g[300] = math.nan, math.inf, -math.inf
        g[512:640] = 1e30
        g[640:768] *= 1e-30
        g[768:896] = 0
        g[900] = 1e18
        for _ in range(2):
            p.grad = g.cuda()
            was = before(opt, p, bits)
            opt.step()
            m, v = opt.moments()[0]
            if bits == 32:
                nan = torch.isnan(m).cpu()
                assert nan[5] and m[200].item() == math.inf and m[300].item() == -math.inf and nan.sum() == 1
                assert torch.isinf(v[512:640]).all()
            else:
                m32, v32 = orc.moments32(g, *was[1:3], (0.9, 0.999))
                rm, rv = orc.noise(1280, was[3] + 1, 0)
                for got, x, r, form in ((m, m32, rm, (14, False)), (v, v32, rv, (30, True))):
                    codes, exps = orc.moment_codes(x, r, *form)
                    want = orc.moment_values(codes, exps, *form, 1280)
                    got = got.cpu().double()
                    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
            assert torch.isfinite(p[384:512]).all() and (bits == 32 or (p[768:896] == 0).all())


def test_codes_keep_the_mean():
    """Without gradients v loses a thousandth a step, far below its unit: the mean over many elements follows the formula. A code's rounding has
    a variance of at most a quarter of its unit's square (unit at most an eighth of the value): after n steps at most n / 256 of the value's square
    an element, in the sum over N elements sqrt(n / 256 / N) of it: 5 of those, and 2^-17 of the unit a step for the noise's 16 bits."""
    import kernels
    N, n = 1 << 17, 300
    p = torch.zeros(N, device="cuda")
    opt = kernels.AdamW([p], lr=0.0, betas=(0.9, 0.999), state_bits=8, weight_decay=0.0)
    p.grad = torch.exp(torch.randn(N, generator=torch.Generator().manual_seed(7))).cuda()
    opt.step()
    start = opt.moments()[0][1].double().sum()
    p.grad = torch.zeros(N, device="cuda")
    for _ in range(n):
        opt.step()
    got = (opt.moments()[0][1].double().sum() / start).item()
    v = opt.moments()[0][1].double()
    spread = math.sqrt(N * (v * v).mean().item()) / v.mean().item() / N  # of a sum of N such values, relative, where each is off by its own size
    assert abs(got / 0.999 ** n - 1) < 5 * math.sqrt(n / 256) * spread + n * 2.0 ** -20
    assert got < 0.8


def test_next_to_torch():
    """The same as torch's optimizer over a few steps: float32 roundings of the same formula (each step within 32 half steps of its update, and
    2 of the parameter)."""
    import kernels
    params, grads = make([(257, 33), (100,)], F, 8)
    mine, theirs = params, [p.detach().clone().requires_grad_(True) for p in params]
    a = kernels.AdamW(mine, lr=1e-3, weight_decay=0.05)
    b = torch.optim.AdamW(theirs, lr=1e-3, weight_decay=0.05)
    for n in range(1, 8):
        for p, q, g in zip(mine, theirs, grads()):
            p.grad, q.grad = g.cuda(), g.cuda()
        a.step(), b.step()
        for p, q in zip(mine, theirs):
            # an update is at most lr / (1 - beta1) / sqrt(1 - beta2)-ish; in these first steps below 4 lr
            assert ((p - q).abs() <= n * (2 * 2 * orc.EPS32 * q.abs() + 2 * 32 * orc.EPS32 * 4e-3)).all()
    # and from its state
    c = kernels.AdamW(theirs, lr=1e-3, weight_decay=0.05)
    c.load_state_dict(b.state_dict())
    for p in theirs:
        assert int(c.state[p]["step"]) == 7 and c.state[p]["step"].is_cuda
        assert torch.equal(c.state[p]["exp_avg"], b.state[p]["exp_avg"])


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dicts(bits):
    import kernels
    params, grads = make([(300, 5), (77,)], BF, 9)
    opt = kernels.AdamW(params, state_bits=bits, seed=5)
    for _ in range(2):
        for p, g in zip(params, grads()):
            p.grad = g.cuda()
        opt.step()
    others = [p.detach().clone().requires_grad_(True) for p in params]
    other = kernels.AdamW(others, state_bits=bits, lr=0.5)
    saved = copy.deepcopy(opt.state_dict())
    other.load_state_dict(saved)
    again = copy.deepcopy(opt)
    for p, q, g in zip(params, others, grads()):
        p.grad, q.grad = g.cuda(), g.cuda()
    for p, r in zip(params, again.param_groups[0]["params"]):
        r.grad = p.grad.clone()
    for o in (opt, other, again):
        o.step()
    for p, q, r in zip(params, others, again.param_groups[0]["params"]):
        assert torch.equal(p, q) and torch.equal(p, r)
        for k, t in opt.state[p].items():
            assert t.dtype == other.state[q][k].dtype and torch.equal(t, other.state[q][k])
    # what was loaded is a copy
    assert all(int(saved["state"][k]["step"]) == 2 for k in saved["state"])
    with pytest.raises(ValueError, match="bits"):
        kernels.AdamW(others, state_bits=40 - bits).load_state_dict({**saved, "param_groups": [{**saved["param_groups"][0], "state_bits": 40 - bits}]})


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    import kernels
    params, grads = make([(500,), (129, 3)], F, 10)
    twins = [p.detach().clone().requires_grad_(True) for p in params]
    lr = torch.tensor(1e-2, device="cuda")
    opt, twin = kernels.AdamW(params, lr=lr, state_bits=bits), kernels.AdamW(twins, lr=1e-2, state_bits=bits)
    static = [torch.zeros_like(p) for p in params]
    for p, s in zip(params, static):
        p.grad = s
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    series = [grads() for _ in range(5)]
    graph = None
    for i, gs in enumerate(series):
        for p, q, s, g in zip(params, twins, static, gs):
            s.copy_(g)
            q.grad = g.cuda()
        if i == 2:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        if i >= 3:
            lr.fill_(1e-3)
            twin.param_groups[0]["lr"] = float(lr)
        if graph is None:
            opt.step()
        else:
            graph.replay()
        twin.param_groups[0]["lr"] = float(lr)
        twin.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q) and int(opt.state[p]["step"]) == i + 1


def test_other_streams_and_autograd_notices():
    import kernels
    p = torch.ones(1000, device="cuda", requires_grad=True)
    opt = kernels.AdamW([p])
    side = torch.cuda.Stream()
    y = (p * p).sum()  # keeps p
    p.grad = torch.ones_like(p)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    assert (p < 1).all()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_moments_into_given_tensors():
    import kernels
    params, grads = make([(1000,), (3, 129)], F, 11)
    opt = kernels.AdamW(params, state_bits=8)
    for p, g in zip(params, grads()):
        p.grad = g.cuda()
    opt.step()
    flat = torch.full((2, 1400), 7.0, device="cuda")
    out = [(flat[0, 1:1001], flat[1, 1:1001]), (flat[0, 1003:1390].view(3, 129), flat[1, 1003:1390].view(3, 129))]
    opt.moments(out=out)
    for (a, b), (c, d) in zip(out, opt.moments()):
        assert torch.equal(a, c) and torch.equal(b, d)
    assert (flat[:, 0] == 7).all() and (flat[:, 1001:1003] == 7).all() and (flat[:, 1390:] == 7).all()
