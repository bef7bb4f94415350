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


def test_fp8_refusals():
    import kernels
    from torch.autograd import forward_ad
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    rows = kernels.Fp8Rows(torch.zeros(4, 8).to(torch.float8_e4m3fn), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8))
    for call in (lambda: kernels.fp8_linear(x, w), lambda: kernels.fp8_linear(x, rows), lambda: kernels.quantize_fp8(x), lambda: kernels.fp8_linear(rows, rows)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.func.vmap(lambda t: call())(x)
    for bad in (lambda: kernels.fp8_linear(x.double(), w), lambda: kernels.fp8_linear(x, w.double())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(ValueError):
        kernels.fp8_linear(rows, w)
    with pytest.raises(ValueError):
        kernels.fp8_linear(x, w, check_timeout=True)
    wants = torch.zeros(2, 8, requires_grad=True)
    for call in (lambda: kernels.fp8_linear(wants, rows), lambda: kernels.fp8_linear(x, rows, torch.zeros(4, requires_grad=True)),
                 lambda: kernels.quantize_fp8(wants)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(2, 8), torch.ones(2, 8))
        for call in (lambda: kernels.fp8_linear(dual, w), lambda: kernels.quantize_fp8(dual), lambda: kernels.fp8_linear(dual, rows)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()


def test_fp8_abi():
    import flb_native as nat
    L = nat.lib
    assert L.flb_fp8_exps_bytes(1, 1) == 512 and L.flb_fp8_exps_bytes(129, 513) == 2048 and L.flb_fp8_exps_bytes(0, 5) == 0

    def rows(x=16, ldx=8, codes=16, exps=16, R=1, K=8, dtype=0):
        return L.flb_fp8_rows(x, ldx, codes, exps, R, K, dtype, None)

    assert rows(dtype=5) == 2 and rows(R=-1) == 1 and rows(K=0) == 1 and rows(K=1 << 31) == 6 and rows(R=1 << 40) == 1
    assert rows(x=None) == 1 and rows(ldx=-1) == 1 and rows(codes=24) == 3 and rows(exps=8) == 3 and rows(x=18) == 3 and rows(R=0, x=None) == 0

    def rows2(bias=None, ws=None, n=0, codes_t=16, R=3, C=5, bias_dtype=0):
        return L.flb_fp8_rows2(16, 8, 16, 16, codes_t, 16, bias, bias_dtype, R, C, 0, ws, n, None)

    assert rows2(codes_t=None) == 1 and rows2(codes_t=24) == 3 and rows2(bias=16) == 8 and rows2(bias=16, ws=16, n=19) == 8
    assert rows2(bias=16, ws=8, n=64) == 3 and rows2(bias=16, bias_dtype=4) == 2 and rows2(R=0) == 0 and rows2(C=0) == 1

    def linear(x=16, ldx=8, xc=None, ldc=0, xe=None, wc=16, ldw=16, we=16, out=16, M=4, N=8, K=8, ws=256, n=1 << 30, dtype=2, bias=None, bias_dtype=0):
        return L.flb_fp8_linear(x, ldx, xc, ldc, xe, wc, ldw, we, bias, bias_dtype, out, M, N, K, dtype, ws, n, 0, None)

    assert linear(dtype=3) == 2 and linear(bias=16, bias_dtype=9) == 2 and linear(K=0) == 1 and linear(M=-1) == 1 and linear(M=0, x=None) == 0
    assert linear(x=None) == 1 and linear(xc=16) == 1 and linear(x=None, xc=16, ldc=16) == 1 and linear(wc=None) == 1 and linear(out=None) == 1
    assert linear(ldw=4) == 1 and linear(ldw=24) == 3 and linear(wc=8) == 3 and linear(we=8) == 3 and linear(out=17) == 3
    assert linear(x=None, xc=16, ldc=4, xe=16) == 1 and linear(x=None, xc=16, ldc=24, xe=16) == 3
    assert linear(ws=None) == 8 and linear(n=100) == 8 and linear(ws=128) == 3 and linear(M=1 << 30, N=1 << 30) == 1
    assert L.flb_fp8_linear_workspace_bytes(1 << 30, 1 << 30, 8, 0) == 0
    for drop, limit in ((-2, 1), (0, 0), (1 << 40, 1)):
        assert L.flb_fp8_linear_wait_test(16, 8, None, 0, None, 16, 16, 16, None, 0, 16, 4, 8, 8, 2, 256, 1 << 30, 1, drop, limit, None) == 1
