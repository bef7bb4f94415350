"""The row operators inside the FLB model: blocks with fused norms and gates, the whole-grid training path with its
intermediates in 8 bits, and decoding with an 8-bit head."""
import pytest
import torch
import torch.nn.functional as F

from test_flb_model import _bf16_model, _max_rel, _train_grads

pytestmark = pytest.mark.gpu


def _fp32_model(c, cuda, **kw):
    from flb_model import FLBTransformer
    return FLBTransformer(c["vocab"], hidden_dim=c["hidden"], num_layers=c["layers"], seq_len=c["seq_len"], batch_size=c["batch"],
                          **kw).to(cuda)


def _loss(m, g, cuda):
    c = g["config"]
    logits, aux, _ = m(g["tokens"].to(cuda))
    return logits, aux, F.cross_entropy(logits.reshape(-1, c["vocab"]), g["targets"].to(cuda).reshape(-1)) + aux


def test_fused_model_matches_reference(cuda, flb_golden):
    """The model with fused norms and gates (float32, per-tick path: the operators under vmap and vjp) against the
    reference's outputs and gradients, at the bounds of the model without them."""
    g = flb_golden
    m = _fp32_model(g["config"], cuda, fused_ops=True)
    m.load_state_dict(g["state_dict"], strict=True)
    m.eval()
    logits, aux, loss = _loss(m, g, cuda)
    assert torch.allclose(logits.cpu(), g["logits"], atol=2e-3)
    assert abs(aux.item() - g["aux_loss"].item()) < 2e-3 * max(1.0, g["aux_loss"].abs().item())
    loss.backward()
    for k, p in m.named_parameters():
        if k not in g["grads"]:
            assert p.grad is None or not p.grad.any(), k
            continue
        ref = g["grads"][k]
        assert (p.grad.cpu() - ref).abs().max().item() <= 2e-3 * max(ref.abs().max().item(), 1e-3), k


class _PlainNorm(torch.autograd.Function):
    """LayerNorm whose backward reads the kept form of its normalised rows, in torch operations."""
    generate_vmap_rule = True

    @staticmethod
    def forward(x, w, b):
        mean = x.mean(-1, keepdim=True)
        rs = torch.rsqrt(((x - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
        h = (x - mean) * rs
        return h * w + b, _plain_kept(h), rs

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.mark_non_differentiable(*output[1:])
        ctx.save_for_backward(inputs[1], *output[1:])

    @staticmethod
    def backward(ctx, dy, *_):
        w, h, rs = ctx.saved_tensors
        gw = dy * w
        dx = rs * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
        axes = tuple(range(dy.ndim - 1))
        return dx, (dy * h).sum(axes), dy.sum(axes)


class _PlainGate(torch.autograd.Function):
    generate_vmap_rule = True

    @staticmethod
    def forward(x, z):
        return x * torch.sigmoid(z), _plain_kept(x), _plain_kept(z)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.mark_non_differentiable(*output[1:])
        ctx.save_for_backward(*output[1:])

    @staticmethod
    def backward(ctx, dy, *_):
        x, z = ctx.saved_tensors
        g = torch.sigmoid(z)
        return dy * g, dy * x * g * (1 - g)


def _plain_kept(x):
    """The kept form of rows of at most 128 elements."""
    assert x.shape[-1] <= 128
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    unit = torch.exp2((e - 7 + (m >= 127.5 / 128)).clamp(min=-126).to(x.dtype))
    return torch.round(x / unit) * unit


def test_kept_model_matches_plain_kept_model(cuda, flb_golden, monkeypatch):
    """keep8: the same outputs as without it, and the gradients of the same network built from torch operations
    that keep the same 8-bit values (the per-tick path's bound for float32)."""
    import flb_model.model as fm
    g = flb_golden
    assert g["config"]["hidden"] <= 128
    m = _fp32_model(g["config"], cuda, fused_ops=True, keep8=True)
    m.load_state_dict(g["state_dict"])
    m.eval()
    logits, _, loss = _loss(m, g, cuda)
    assert torch.allclose(logits.cpu(), g["logits"], atol=2e-3)
    loss.backward()
    got = {k: p.grad.clone() for k, p in m.named_parameters() if p.grad is not None}
    m.zero_grad(set_to_none=True)
    monkeypatch.setattr(fm, "sigmoid_gate", lambda x, z, keep8: _PlainGate.apply(x, z)[0])
    monkeypatch.setattr(fm.FusedLayerNorm, "forward", lambda self, x: _PlainNorm.apply(x, self.weight, self.bias)[0])
    _loss(m, g, cuda)[2].backward()
    for k, p in m.named_parameters():
        if p.grad is None:
            assert k not in got
            continue
        assert (got[k] - p.grad).abs().max().item() <= 2e-3 * max(p.grad.abs().max().item(), 1e-3), k


def test_fused_model_arguments():
    from flb_model import FLBTransformer
    with pytest.raises(ValueError, match="keep8 needs fused_ops"):
        FLBTransformer(10, hidden_dim=64, num_layers=2, seq_len=4, batch_size=2, keep8=True)


UNITS = (1, 1, 1, 3, 1, 1, 9, 3, 3, 9, 1, 1, 1, 1)  # rows of d_model a cell and batch row has in each bf16 plane


@pytest.mark.parametrize("D,L,S,B,H", [(64, 4, 6, 3, 8), (80, 3, 7, 5, 8), (768, 4, 5, 16, 12)])
def test_whole_grid_training_in_8_bits(cuda, D, L, S, B, H):
    """engine.native_flb_save = "int8": the outputs of the forward without it, a buffer of a quarter of the bf16 planes'
    size, and the gradients that the bf16 path gives when its kept intermediates are replaced by what their
    kept form stands for (2e-2 of the largest magnitude, the bound between the bf16 paths)."""
    import flb_native as nat
    import kernels
    from wavefront import flb_cells
    m = _bf16_model(29, D=D, L=L, S=S, B=B, heads=H)
    tok = torch.randint(0, 50, (B, S), device=cuda)
    targets = torch.randint(0, 50, (B, S), device=cuda)
    m.engine.native_flb_save = "int8"
    g8, l8 = _train_grads(m, tok, targets, True)
    ws = m.engine.graph_workspace
    kept = ws["flb_saved8"]
    rows = L * S * B * 18
    assert kept.numel() <= rows * D + 256 + rows * -(-D // 128) and "flb_saved" not in ws
    m.engine.native_flb_save = True
    calls = []

    def rounded(engine, w, grad_grids, saved=None):
        planes, at = saved.view(torch.bfloat16), 0
        for p, u in enumerate(UNITS):
            n = u * L * S * B * D
            if 2 <= p <= 7:
                v = planes[at:at + n].view(-1, D)
                v.copy_(kernels.unpack8(kernels.pack8(v)))
            at += n
        assert at == planes.numel()
        calls.append(p)
        return backward(engine, w, grad_grids, saved)

    backward = flb_cells.native_flb_backward
    flb_cells.native_flb_backward = rounded
    try:
        gb, lb = _train_grads(m, tok, targets, True)
    finally:
        flb_cells.native_flb_backward = backward
    assert calls and abs(l8 - lb) <= 2e-2 * abs(lb)
    assert set(g8) == set(gb)
    for k in gb:
        assert _max_rel(g8[k], gb[k]) < 2e-2, (k, _max_rel(g8[k], gb[k]))
    m.engine.native_flb_save = "bf8"
    with pytest.raises(ValueError, match="native_flb_save"):
        _train_grads(m, tok, targets, True)


def test_whole_grid_training_in_8_bits_graphed(cuda):
    """The same captured as CUDA graphs: the eager path's loss and gradients over two steps with new weights."""
    ma, mb = _bf16_model(31, D=128), _bf16_model(31, D=128)
    for m in (ma, mb):
        m.engine.native_flb_save = "int8"
    tok = torch.randint(0, 50, (3, 6), device=cuda)
    targets = torch.randint(0, 50, (3, 6), device=cuda)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        graphed = mb.engine.graphed(mb.embedding(tok).detach())
    for step in range(2):
        outs = []
        for m, eng in ((ma, None), (mb, graphed)):
            m.zero_grad(set_to_none=True)
            with torch.autocast("cuda", dtype=torch.bfloat16):
                logits, aux, _ = m(tok, engine=eng)
            loss = F.cross_entropy(logits.float().reshape(-1, 50), targets.reshape(-1)) + aux
            loss.backward()
            outs.append((loss.item(), {k: p.grad.float().clone() for k, p in m.named_parameters() if p.grad is not None}))
        (la, ga), (lb, gb) = outs
        assert abs(la - lb) <= 1e-3 * abs(la) and set(ga) == set(gb)
        for k in ga:
            assert _max_rel(gb[k], ga[k]) < 1e-2, (step, k)
        with torch.no_grad():
            for pa, pb in zip(ma.parameters(), mb.parameters()):
                pa.mul_(0.95)
                pb.mul_(0.95)


def test_decode_with_8_bit_head(cuda):
    """greedy_decode with the head in 8-bit integers: graphed and eager give the tokens of a loop that takes the
    last state through int8_linear."""
    import kernels
    from flb_model import greedy_decode
    m = _bf16_model(37, S=8, B=2, D=64, V=777)
    head = kernels.Int8Linear.from_linear(m.head)
    prompt = torch.randint(0, 777, (2, 8), device=cuda)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a = greedy_decode(m, prompt, 5, graphed=False, head=head)
        b = greedy_decode(m, prompt, 5, graphed=True, head=head)
    assert torch.equal(a, b)
    window = prompt.clone()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        for s in range(5):
            y = m.engine(m.embedding(window), {})[0].view(4, 8, 2, 64)[-1].transpose(0, 1)
            nxt = kernels.int8_linear(y[:, -1].contiguous(), kernels.Int8Rows(head.codes, head.scale), head.bias.float()).argmax(-1)
            assert torch.equal(nxt, a[:, s])
            window = torch.cat([window[:, 1:], nxt[:, None]], dim=1)
