"""What the choice of a token and AdamW refuse, before any GPU is needed."""
import ctypes

import pytest
import torch


def test_sample_refusals():
    import kernels
    x, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kernels.sample(x, u)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        kernels.sample(x.double(), u)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.vmap(lambda t: kernels.sample(t, u[0]))(x)
    with pytest.raises(TypeError):
        kernels.sample(x, u, top_k=2.5)


def test_sample_abi():
    import flb_native as nat

    def call(logits=16, u=16, token=16, rows=1, V=8, dtype=0, ld=8, t=None, k=None):
        return nat.lib.flb_sample(logits, ld, u, 0, token, rows, V, dtype, t, 1.0, k, 0, None, 1.0, None, 0.0, None)

    assert call(dtype=7) == 2 and call(V=0) == 1 and call(rows=-1) == 1 and call(V=262145) == 6 and call(ld=-1) == 1
    assert call(logits=None) == 1 and call(u=None) == 1 and call(token=None) == 1
    assert call(logits=18) == 3 and call(token=12) == 3 and call(t=2) == 3 and call(k=12) == 3
    assert call(rows=0, logits=None) == 0 and call(rows=1 << 40) == 1


def test_adamw_refusals():
    import kernels
    p = torch.zeros(4, requires_grad=True)
    for bad in ({"lr": -1.0}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"eps": -1e-8}, {"weight_decay": -1.0}, {"state_bits": 16},
                {"lr": torch.zeros(2)}):
        with pytest.raises(ValueError):
            kernels.AdamW([p], **bad)
    with pytest.raises(TypeError):
        kernels.AdamW([torch.zeros(4, dtype=torch.float64, requires_grad=True)])
    with pytest.raises(ValueError):
        kernels.AdamW([p, p])
    opt = kernels.AdamW([p])
    opt.step()  # no gradient, nothing to do
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        opt.step()
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.zeros(2, requires_grad=True)], "state_bits": 4})
    assert len(opt.param_groups) == 1 and opt.moments() == []


def test_adamw_abi():
    import flb_native as nat

    def call(dtype=0, bits=32, b1=0.9, b2=0.9, counter=16, count=1, **fields):
        t = nat.AdamWTensor(**{**dict(p=16, g=16, m=16, v=16, m_exps=16, v_exps=16, step=16, n=8), **fields})
        return nat.lib.flb_adamw(ctypes.byref(t), count, dtype, bits, 0.1, None, b1, b2, 1e-8, 0.0, 0, counter, None)

    assert call(dtype=9) == 2 and call(bits=16) == 6 and call(b1=1.0) == 6 and call(b2=-0.5) == 6 and call(b1=float("nan")) == 6
    assert call(count=-1) == 1 and call(n=-1) == 1 and call(n=1 << 50) == 1 and call(p=None) == 1 and call(step=None) == 1 and call(v=None) == 1
    assert call(bits=8, m_exps=None) == 1 and call(p=18) == 3 and call(m=18) == 3 and call(step=20) == 3
    assert call(counter=None) == 8 and call(counter=18) == 3
    assert call(count=0) == 0
    assert nat.lib.flb_adamw_moments(None, 0, None) == 0 and nat.lib.flb_adamw_moments(None, 1, None) == 1
