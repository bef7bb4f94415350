"""Weights kept in 8-bit floating point as they are saved and loaded."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F = torch.float32


def litter(nbytes):
    """Memory of that size that was last used for something else: what the next tensor of the size is likely to get."""
    torch.full((nbytes,), 0xA5, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, F])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 768), (5, 129), (128, 512), (127, 513), (129, 640), (300, 1000), (256, 1024), (33, 2048)])
def test_the_same_rows_have_the_same_bytes(R, K, dtype):
    """All of them, also where no block is: two checkpoints of a weight are equal."""
    import kernels
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(R)).to(dtype).cuda()
    first = kernels.quantize_fp8(x)
    blocks, quads = -(-K // 128), -(-K // 512)
    for _ in range(2):
        litter(first.exps.numel()), litter(R * -(-K // 16) * 16)
        again = kernels.quantize_fp8(x)
        assert torch.equal(again.exps, first.exps) and torch.equal(again.codes.view(torch.uint8), first.codes.view(torch.uint8))
        # [groups, quads, r % 32, r / 32 % 4, b % 4] as rows and blocks
        by_row = again.exps.permute(0, 3, 2, 1, 4).reshape(-1, quads * 4)
        assert (by_row[:R, :blocks] > 0).all() and not by_row[R:].any() and not by_row[:, blocks:].any()


@pytest.mark.parametrize("K,N", [(100, 40), (768, 1000), (1024, 130)])
@pytest.mark.parametrize("bias", [True, False])
def test_a_kept_map_through_a_saved_state(K, N, bias, tmp_path):
    """Saved, and loaded into the map of another weight, on the GPU and through the CPU: the same outputs to the bit."""
    import kernels
    linear = kernels.Fp8Linear(K, N, bias).cuda()
    kept, again = linear.kept(), linear.kept()
    for name, t in kept.state_dict().items():
        other = again.state_dict()[name]
        assert torch.equal(t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t, other.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else other)
    assert set(kept.state_dict()) == ({"codes", "exps", "bias"} if bias else {"codes", "exps"})
    torch.save(kept.state_dict(), tmp_path / "kept.pt")
    x = torch.randn(7, K, device="cuda")
    want = kept(x)
    for where in ("cuda", "cpu"):
        other = kernels.Fp8Linear(K, N, bias).cuda().kept()
        assert not torch.equal(other(x), want)
        other.load_state_dict(torch.load(tmp_path / "kept.pt", map_location=where, weights_only=True))
        assert torch.equal(other(x), want)
        assert torch.equal(other.cpu().cuda()(x), want)
