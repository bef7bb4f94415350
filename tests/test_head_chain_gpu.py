"""The operators around a model's head together, as a training step and a decoding loop use them: the head's product in 8-bit
floating point, AdamW, and the choice of tokens."""
import pytest
import torch
import torch.nn.functional as F

from oracle import head as orc
from test_adamw_gpu import before, check
from test_fp8_linear_gpu import close

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _model(seed, V=777, D=64, L=3, S=8, B=2, **kw):
    from flb_model import FLBTransformer
    torch.manual_seed(seed)
    return FLBTransformer(V, hidden_dim=D, num_layers=L, seq_len=S, batch_size=B, num_heads=8, **kw).cuda().eval()


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(bits):
    """Logits and the head's gradients are fp8_linear's of the states that reach it, the other parameters' gradients come from its
    gradient of those, and AdamW steps them all."""
    import kernels
    m = _model(1, fp8_head=True)
    plain = _model(1)
    assert list(m.state_dict()) == list(plain.state_dict())
    opt = kernels.AdamW(m.parameters(), lr=1e-3, state_bits=bits)
    seen = {}
    m.head.register_forward_hook(lambda mod, args, out: seen.update(top=args[0], logits=out) or args[0].retain_grad())
    tok, targets = torch.randint(0, 777, (2, 8), device="cuda"), torch.randint(0, 777, (2, 8), device="cuda")
    for _ in range(2):
        opt.zero_grad(set_to_none=True)
        logits, aux, _ = m(tok)
        logits.retain_grad()
        (F.cross_entropy(logits.reshape(-1, 777), targets.reshape(-1)) + aux).backward()
        top, w, b, dy = (t.detach().cpu() for t in (seen["top"], m.head.weight, m.head.bias, logits.grad))
        rows, dy = top.reshape(16, 64), dy.reshape(16, 777)
        close(logits.reshape(16, 777), *orc.fp8_product(rows, w, b, torch.float32))
        close(m.head.weight.grad, *orc.fp8_product(dy.t(), rows.t(), None, torch.float32))
        close(seen["top"].grad.reshape(16, 64), *orc.fp8_product(dy, w.t(), None, torch.float32))
        assert m.embedding.weight.grad.abs().sum() > 0
        was = {k: before(opt, p, bits) for k, p in m.named_parameters()}
        grads = {k: p.grad.cpu() for k, p in m.named_parameters() if p.grad is not None}
        opt.step()
        for k, p in m.named_parameters():
            if k in grads:
                check(opt, p, was[k], grads[k], bits)
        seen.clear()


def test_under_autocast_with_the_native_engine():
    """bf16 autocast: the whole-grid kernels below the head. The loss and the gradients of the layers are those of the same model with a plain head to
    what 8 bits allow: a state or weight is off by at most 1/16, a logit's or gradient's relative error in norm is less."""
    m, plain = _model(2, fp8_head=True), _model(2)
    tok, targets = torch.randint(0, 777, (2, 8), device="cuda"), torch.randint(0, 777, (2, 8), device="cuda")
    grads = []
    for x in (m, plain):
        with torch.autocast("cuda", dtype=BF):
            logits, aux, _ = x(tok)
        assert logits.dtype == BF
        (F.cross_entropy(logits.float().reshape(-1, 777), targets.reshape(-1)) + aux).backward()
        grads.append({k: p.grad.float() for k, p in x.named_parameters() if p.grad is not None})
    assert set(grads[0]) == set(grads[1])
    for k in ("head.weight", "head.bias", "embedding.weight"):
        assert (grads[0][k] - grads[1][k]).norm() <= grads[1][k].norm() / 8, k


def test_sample_decode():
    """Graphed and eager decoding give the tokens of a loop over kernels.sample, with the model's head and with one kept in 8 bits."""
    import kernels
    from flb_model import greedy_decode, sample_decode
    m = _model(3, fp8_head=True)
    prompt = torch.randint(0, 777, (2, 8), device="cuda")
    u = torch.rand(6, 2, device="cuda")
    settings = {"temperature": 0.9, "top_k": 100, "top_p": 0.95, "min_p": 0.001}
    for head in (None, m.head.kept(), kernels.Int8Linear.from_linear(m.head)):
        with torch.autocast("cuda", dtype=BF):
            a = sample_decode(m, prompt, u, **settings, graphed=False, head=head)
            b = sample_decode(m, prompt, u, **settings, head=head)
        assert torch.equal(a, b)
        window = prompt.clone()
        with torch.no_grad(), torch.autocast("cuda", dtype=BF):
            for s in range(6):
                logits = m(window)[0][:, -1] if head is None else m(window, head=lambda top: head(top[:, -1]))[0]
                nxt = kernels.sample(logits, u[s], **settings)
                assert torch.equal(nxt, a[:, s]) and torch.equal(nxt.cpu(), orc.sample(logits.cpu(), u[s].cpu(), **settings))
                window = torch.cat([window[:, 1:], nxt[:, None]], dim=1)
        with torch.autocast("cuda", dtype=BF):
            assert torch.equal(sample_decode(m, prompt, u, temperature=0, head=head), greedy_decode(m, prompt, 6, head=head))


def test_a_sequence_without_a_token():
    from flb_model import sample_decode
    m = _model(4)
    prompt = torch.randint(0, 777, (2, 8), device="cuda")

    def head(top):
        logits = m.head(top)
        logits[1] = float("nan")
        return logits

    out = sample_decode(m, prompt, torch.rand(3, 2, device="cuda"), graphed=False, head=head)
    assert (out[1] == -1).all() and (out[0] >= 0).all()


def test_a_captured_training_step_of_the_head():
    """Product, loss, gradients and step as one graph, replayed: the eager steps' parameters."""
    import kernels
    linear = torch.nn.Linear(96, 500).cuda()
    twin = torch.nn.Linear(96, 500).cuda()
    twin.load_state_dict(linear.state_dict())
    a, b = kernels.Fp8Linear.from_linear(linear), kernels.Fp8Linear.from_linear(twin)
    oa, ob = kernels.AdamW(a.parameters(), lr=1e-2, state_bits=8), kernels.AdamW(b.parameters(), lr=1e-2, state_bits=8)
    x, targets = torch.randn(64, 96, device="cuda"), torch.randint(0, 500, (64,), device="cuda")

    def step(m, o):
        o.zero_grad(set_to_none=False)
        F.cross_entropy(m(x), targets).backward()
        o.step()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, oa)
    torch.cuda.current_stream().wait_stream(side)
    step(b, ob)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, oa)
    for i in range(4):
        x.copy_(torch.randn(64, 96, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        step(b, ob)
        assert torch.equal(a.weight, b.weight) and torch.equal(a.bias, b.bias)


def test_one_vector():
    """x without leading axes, forward and backward."""
    import kernels
    x, w = torch.randn(130, device="cuda", requires_grad=True), torch.randn(70, 130, device="cuda", requires_grad=True)
    y = kernels.fp8_linear(x, w)
    dy = torch.randn(70, device="cuda")
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xc, wc, dyc = (t.detach().cpu() for t in (x, w, dy))
    assert y.shape == (70,) and dx.shape == (130,)
    close(y[None], *orc.fp8_product(xc[None], wc, None, torch.float32))
    close(dx[None], *orc.fp8_product(dyc[None], wc.t(), None, torch.float32))
    close(dw, *orc.fp8_product(dyc[:, None], xc[:, None], None, torch.float32))


def test_calls_on_two_streams_at_once():
    """Products, choices and steps on two streams, each with what it needs of its own."""
    import kernels
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [torch.randn(300, 640, device="cuda") for _ in range(2)]
    ws = [kernels.quantize_fp8(torch.randn(500, 640, device="cuda")) for _ in range(2)]
    us = [torch.rand(300, device="cuda") for _ in range(2)]
    ps = [torch.randn(5000, device="cuda") for _ in range(2)]
    opts = [kernels.AdamW([p], state_bits=8) for p in ps]
    for p in ps:
        p.grad = torch.ones_like(p)
    twins = [p.clone() for p in ps]
    want = [kernels.sample(kernels.fp8_linear(x, w), u, top_p=0.7) for x, w, u in zip(xs, ws, us)]
    for t in twins:
        o = kernels.AdamW([t], state_bits=8)
        t.grad = torch.ones_like(t)
        for _ in range(20):
            o.step()
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = kernels.sample(kernels.fp8_linear(xs[i], ws[i]), us[i], top_p=0.7)
                opts[i].step()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], want[i]) and torch.equal(ps[i], twins[i])


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_device_than_the_current_one():
    import kernels
    with torch.cuda.device(0):
        x = torch.randn(40, 200, device="cuda:1", requires_grad=True)
        w = torch.randn(90, 200, device="cuda:1", requires_grad=True)
        y = kernels.fp8_linear(x, w)
        y.sum().backward()
        token = kernels.sample(y.detach(), torch.rand(40, device="cuda:1"))
        opt = kernels.AdamW([w])
        opt.step()
    assert token.device == y.device == x.grad.device == w.device
    with pytest.raises(ValueError, match="different devices"):
        kernels.sample(y.detach(), torch.rand(40, device="cuda:0"))
