"""More refusals of the row operators and 8-bit products, and what their modules do without a kernel (no GPU,
but for the test that is marked)."""
import pytest
import torch
from torch.autograd import forward_ad


def test_wait_test_arguments():
    import flb_native as nat
    assert nat.lib.flb_selftest_late_copy(16, 16, 8, 0, None) == 1 and nat.lib.flb_selftest_late_copy(16, 16, 16, 100001, None) == 1
    assert nat.lib.flb_selftest_late_copy(16, 24, 16, 0, None) == 3
    assert nat.lib.flb_int8_linear_wait_test(16, 64, None, 0, None, 16, 64, 16, None, 0, 16, 4, 8, 64, 2, 256, 1 << 30, 1, -2, 1, None) == 1
    assert nat.lib.flb_int8_linear_wait_test(16, 64, None, 0, None, 16, 64, 16, None, 0, 16, 4, 8, 64, 2, 256, 1 << 30, 1, 0, 0, None) == 1


def int8_rows(n=4, K=8, requires_grad=False):
    import kernels
    return kernels.Int8Rows(torch.ones(n, K, dtype=torch.int8), torch.ones(n, requires_grad=requires_grad), torch.float32)


def calls():
    """Every operator that reads floating-point tensors, as functions of one of them (the others have no derivative)."""
    import kernels
    x, w = torch.ones(2, 8), torch.ones(8)
    return [kernels.layer_norm, lambda t: kernels.layer_norm(x, t[0]), lambda t: kernels.layer_norm(x, None, t[0]),
            lambda t: kernels.layer_norm(t, w, w, keep8=True), lambda t: kernels.sigmoid_gate(t, x), lambda t: kernels.sigmoid_gate(x, t),
            kernels.layer_norm_int8, lambda t: kernels.layer_norm_int8(x, t[0]), kernels.quantize_int8,
            lambda t: kernels.int8_linear(t, int8_rows()), lambda t: kernels.int8_linear(x, int8_rows(2), t[:, 0])]


def test_tangents_are_refused():
    for call in calls():
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.ones(2, 8), torch.ones(2, 8))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(dual)
            # without its tangent the call goes on to the check of its device
            with pytest.raises(RuntimeError, match="CUDA tensors only"):
                call(forward_ad.unpack_dual(dual).primal)


def test_scales_that_want_a_gradient_are_refused():
    """The scales of integer rows are inputs of the product like any other."""
    import kernels
    x, wants = torch.ones(2, 8), int8_rows(requires_grad=True)
    for call in (lambda: kernels.int8_linear(x, wants), lambda: kernels.int8_linear(wants, int8_rows())):
        with pytest.raises(RuntimeError, match="has no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_check_timeout_reaches_the_kernel(monkeypatch):
    import sys
    import kernels

    class Ops:
        calls = []

        @staticmethod
        def int8_linear(*args):
            Ops.calls.append(args[-1])

        @staticmethod
        def quantize_int8(w):
            return int8_rows()[:2]

    monkeypatch.setattr(sys.modules["kernels.int8_linear"], "flb_ops", Ops)
    x, linear = torch.ones(2, 8), torch.nn.Linear(8, 4)
    for check in (True, False):
        kernels.int8_linear(x, int8_rows(), check_timeout=check)
        kernels.int8_linear(int8_rows(), int8_rows(), None, check)
        kernels.Int8Linear(int8_rows(), check_timeout=check)(x)
        kernels.Int8Linear.from_linear(linear, check)(int8_rows())
        assert Ops.calls == [check] * 4
        Ops.calls.clear()


CASTS = [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.bfloat16().float(),
         lambda m: m.type(torch.float16)]


@pytest.mark.parametrize("cast", CASTS)
def test_a_cast_of_the_module_keeps_the_integers_and_scales(cast):
    import kernels
    rows = kernels.Int8Rows(torch.arange(-16, 16, dtype=torch.int8).reshape(4, 8), torch.rand(4) + 1 / 3)
    m = torch.nn.Sequential(kernels.Int8Linear(rows, torch.ones(4)), torch.nn.Linear(4, 4))
    want = [t.clone() for t in rows[:2]]
    assert cast(m) is m
    for got, t in zip((m[0].codes, m[0].scale), want):
        assert got.dtype == t.dtype and torch.equal(got, t)
    assert m[0].bias.dtype == m[1].weight.dtype and set(m[0].state_dict()) == {"codes", "scale", "bias"}
    m[0].to("meta")
    assert m[0].scale.device.type == m[0].codes.device.type == "meta" and m[0].scale.dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("cast", CASTS)
def test_a_cast_module_gives_the_same(cast):
    import kernels
    linear = torch.nn.Linear(96, 40)
    x = torch.randn(7, 96, device="cuda")
    m = torch.nn.Sequential(kernels.Int8Linear.from_linear(linear.cuda()))
    m[0].bias = None
    want = m(x)
    assert torch.equal(cast(m)(x), want) and torch.equal(m.cpu().cuda()(x), want)


def test_a_head_without_modules_is_a_head():
    """FLBTransformer takes a head that is given, also an empty nn.Sequential, whose length is zero."""
    from flb_model import FLBTransformer
    m = FLBTransformer(11, hidden_dim=8, num_layers=2, seq_len=3, batch_size=2, num_heads=2).eval()
    grids = [torch.randn(6, 2, 8) for _ in range(4)]
    top = grids[0].view(2, 3, 2, 8)[-1].transpose(0, 1)
    assert torch.equal(m.grids_to_outputs(grids, torch.nn.Sequential())[0], top)
    assert torch.equal(m.grids_to_outputs(grids)[0], m.head(top))
