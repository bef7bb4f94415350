"""The choice of a token from logits on a B200, against the definition in 64 bits."""
import math

import pytest
import torch

from oracle import head as orc

pytestmark = pytest.mark.gpu

BF, H, F = torch.bfloat16, torch.float16, torch.float32
LARGEST = 262144


def logits_of(rows, V, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = scale * torch.randn(rows, V, generator=g) + 6 * (torch.rand(rows, V, generator=g) < 10 / V)
    return x.to(dtype), torch.rand(rows, generator=g)


def check(x, u, **settings):
    import kernels
    per_row = {k: torch.tensor(v, dtype=torch.int64 if k == "top_k" else F, device="cuda") if isinstance(v, list) else v for k, v in settings.items()}
    got = kernels.sample(x.cuda(), u.cuda(), **per_row)
    exact = {k: torch.tensor(v, dtype=F).tolist() if isinstance(v, list) and k != "top_k" else v for k, v in settings.items()}
    assert got.dtype == torch.int64 and got.shape == x.shape[:-1]
    assert got.cpu().tolist() == orc.sample(x, u, **exact).tolist()


SETTINGS = [{}, {"temperature": 0}, {"temperature": 0.7, "top_k": 50, "top_p": 0.95}, {"top_k": 1}, {"top_k": 7}, {"top_p": 0.9}, {"top_p": 0.0},
            {"top_p": 1e-9}, {"top_p": 0.999999}, {"min_p": 0.05}, {"min_p": 1.0}, {"temperature": 1.5, "top_k": 300, "top_p": 0.6, "min_p": 0.1},
            {"temperature": 0.01}, {"temperature": 100.0, "top_p": 0.5}, {"temperature": 1e-300}, {"top_k": 10 ** 12, "min_p": 0.01}]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", [BF, H, F])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (5, 17), (4, 1000), (2, 4099), (3, 32000)])
def test_settings(rows, V, dtype, settings):
    x, u = logits_of(rows, V, dtype, rows * V)
    check(x, u, **settings)


@pytest.mark.parametrize("rows", [1, 2, 18, 37, 74, 149, 300, 700])
def test_rows_and_blocks(rows):
    """Each number of blocks a row, and more rows than run at once."""
    x, u = logits_of(rows, 9001, BF, rows)
    check(x, u, temperature=0.8, top_k=100, top_p=0.9)
    check(x, u)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("V", [131071, LARGEST])
def test_large_vocabularies(V, dtype):
    x, u = logits_of(2, V, dtype, V)
    check(x, u, top_p=0.9)
    check(x, u, min_p=0.001, top_k=5000)
    check(x, u, temperature=0)


def test_many_rows_that_need_clusters():
    x, u = logits_of(80, LARGEST, F, 1)
    import kernels
    got = kernels.sample(x.cuda(), u.cuda(), top_p=0.8)
    few = torch.tensor([0, 1, 40, 79])
    assert got.cpu()[few].tolist() == orc.sample(x[few], u[few], top_p=0.8).tolist()


@pytest.mark.parametrize("dtype", [BF, H, F])
def test_masks_and_infinities(dtype):
    x, u = logits_of(9, 5000, dtype, 3)
    x[0] = -math.inf
    x[1, 7] = math.nan
    x[2] = -math.inf
    x[2, 4321] = -2.0
    x[3, [5, 17, 4000]] = math.inf
    x[4, ::2] = -math.inf
    x[5] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).min
    x[6, 100] = torch.finfo(dtype).max
    x[7, 1:] = -math.inf
    x[8, :] = math.nan
    for settings in ({}, {"top_k": 2}, {"top_p": 0.5}, {"temperature": 0}, {"top_k": 3, "top_p": 0.4, "min_p": 0.2}):
        check(x, u, **settings)


@pytest.mark.parametrize("dtype", [BF, H, F])
@pytest.mark.parametrize("V", [1, 37, 1000, 8191])
def test_equal_logits_go_by_index(V, dtype):
    """Equal logits: the distribution function is a staircase, and cuts go to the lowest indices."""
    n = min(V, 64)
    x = torch.full((n, V), -3.25, dtype=dtype)
    x[:, 1::2] = torch.where(torch.rand(n, x[:, 1::2].shape[1], generator=torch.Generator().manual_seed(V)) < 0.5, -3.25, -3.25).to(dtype)
    u = (torch.arange(n).double() + 0.5) / n
    check(x, u)
    check(x, u, top_p=0.5)
    check(x, u, top_k=max(1, V // 3))
    check(x, u, top_k=max(1, V // 3), top_p=0.5)
    check(x, u, temperature=0)
    # two groups of equal ones, cut within the second; zeros of both signs are equal
    x[:, ::3] = 0.0
    x[:, 3::6] = -0.0
    check(x, u, top_k=max(1, V // 2))
    check(x, u, top_p=0.99)
    check(x, u, temperature=0)


def test_close_float32_logits():
    """Logits that differ in their last bits alone: thresholds in the histogram's last level."""
    g = torch.Generator().manual_seed(5)
    x = 1 + torch.randint(0, 700, (16, 3000), generator=g) * 2.0 ** -23
    u = torch.rand(16, generator=g)
    for settings in ({"top_k": 1234}, {"top_p": 0.3}, {"top_k": 1500, "top_p": 0.77}):
        check(x, u, **settings)
    check(x - 2 ** -3, u, top_p=0.51)


def test_the_ends_of_u():
    x, _ = logits_of(6, 2000, F, 8)
    u = torch.tensor([0.0, 1.0, 1 - 2.0 ** -24, 2.0 ** -30, 5.0, -1.0])
    check(x, u)
    check(x, u, top_k=10)
    check(x, u.double(), top_p=0.5)
    import kernels
    odd = torch.tensor([math.nan, math.inf] * 3, device="cuda")
    assert (kernels.sample(x.cuda(), odd) >= 0).all()


def test_a_setting_for_each_row():
    x, u = logits_of(8, 6000, F, 9)
    check(x, u, temperature=[0.0, 0.5, 1.0, 2.0, -1.0, 0.1, 1.0, 1.0], top_k=[0, 5, 0, 6000, 3, 1, -4, 50], top_p=[1.0, 0.9, 0.1, 1.0, 0.5, 0.0, 2.0, 0.7],
          min_p=[0.0, 0.0, 0.2, 0.001, 0.0, 1.0, 0.0, 3.0])
    check(x, u.double(), top_k=[3] * 8)


def test_layouts():
    import kernels
    x, u = logits_of(12, 3001, BF, 10)
    want = orc.sample(x, u, top_p=0.8)
    # last positions of a batch, odd pitches and offsets, columns, leading axes
    wide = torch.zeros(12, 5, 3001, dtype=BF)
    wide[:, -1] = x
    assert torch.equal(kernels.sample(wide.cuda()[:, -1], u.cuda(), top_p=0.8).cpu(), want)
    for at in (1, 3, 8):
        off = torch.zeros(12, 3020, dtype=BF)
        off[:, at:at + 3001] = x
        assert torch.equal(kernels.sample(off.cuda()[:, at:at + 3001], u.cuda(), top_p=0.8).cpu(), want)
    assert torch.equal(kernels.sample(x.cuda().t().contiguous().t(), u.cuda(), top_p=0.8).cpu(), want)
    got = kernels.sample(x.cuda().view(3, 4, 3001), u.cuda().view(3, 4), top_p=0.8)
    assert torch.equal(got.cpu(), want.view(3, 4))
    one = kernels.sample(x[0].cuda(), u[0].cuda(), top_p=0.8)
    assert one.shape == () and int(one) == int(want[0])
    assert kernels.sample(x[:0].cuda(), u[:0].cuda()).shape == (0,)
    # one row for all: a row that is expanded
    rows = x[:1].cuda().expand(12, -1)
    assert torch.equal(kernels.sample(rows, u.cuda()).cpu(), orc.sample(x[:1].expand(12, -1), u))


def test_the_distribution():
    """Tokens over a grid of u come as often as their probability says, to one grid step each side."""
    import kernels
    g = torch.Generator().manual_seed(11)
    x = torch.randn(50, generator=g)
    n = 20000
    u = (torch.arange(n).double() + 0.5) / n
    got = kernels.sample(x.cuda().expand(n, -1), u.cuda(), temperature=0.9, top_k=30, min_p=0.02).cpu()
    tokens, w = orc.kept_tokens(x, temperature=0.9, top_k=30, min_p=0.02)
    counts = torch.bincount(got, minlength=50)
    assert set(got.tolist()) <= set(tokens.tolist())
    assert ((counts[tokens] - n * w / w.sum()).abs() <= 2).all()


def test_captured_and_on_another_stream():
    import kernels
    x, u = logits_of(5, 32000, BF, 12)
    xs, us = x.cuda(), u.cuda()
    want = orc.sample(x, u, top_k=40, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.sample(xs, us, top_k=40, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.sample(xs, us, top_k=40, top_p=0.9)
    y, v = logits_of(5, 32000, BF, 13)
    for a, b in ((x, u), (y, v)):
        xs.copy_(a), us.copy_(b)
        graph.replay()
        assert torch.equal(out.cpu(), orc.sample(a, b, top_k=40, top_p=0.9))
