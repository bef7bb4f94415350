"""Refusals and argument checks of LayerNorm, the 8-bit kept form and the sigmoid gate (no GPU)."""
import pytest
import torch

FLB_SHAPE, FLB_DTYPE, FLB_ALIGN, FLB_UNSUPPORTED, FLB_WORKSPACE = 1, 2, 3, 6, 8
F32, F16, BF16 = 0, 1, 2


def test_cpu_tensors_are_refused():
    import kernels
    x = torch.zeros(2, 8)
    for call in (lambda: kernels.layer_norm(x), lambda: kernels.sigmoid_gate(x, x), lambda: kernels.pack8(x),
                 lambda: kernels.unpack8(kernels.Packed8(torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8),
                                                         torch.Size((2, 8)), torch.float32))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_types_are_refused():
    import kernels
    for t in (torch.float64, torch.int32, torch.complex64):
        x = torch.zeros(2, 8, dtype=t)
        for call in (lambda: kernels.layer_norm(x), lambda: kernels.sigmoid_gate(x, x), lambda: kernels.pack8(x)):
            with pytest.raises(TypeError):
                call()


def test_unpack_checks_its_form():
    import kernels
    codes, exps = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8)
    for bad in (kernels.Packed8(codes, exps, torch.Size((2, 17)), torch.float32), kernels.Packed8(codes, exps, torch.Size((3, 8)), torch.float32),
                kernels.Packed8(codes.t().contiguous().t(), exps, torch.Size((2, 8)), torch.float32),
                kernels.Packed8(codes.float(), exps, torch.Size((2, 8)), torch.float32)):
        with pytest.raises(ValueError):
            kernels.unpack8(bad)


def norm_fwd(x=16, ldx=8, w=None, b=None, wdt=F32, y=16, mean=None, rstd=None, codes=None, exps=None, G=1, R=2, D=8, dt=BF16):
    import flb_native as nat
    return nat.lib.flb_layer_norm_fwd(x, ldx, w, b, wdt, y, mean, rstd, codes, exps, G, R, D, dt, 1e-5, None)


def norm_bwd(x=16, ldx=8, codes=None, exps=None, mean=16, rstd=16, w=None, wdt=F32, dy=16, dx=16, dw=None, db=None, G=1, R=2, D=8,
             dt=BF16, ws=None, n=0):
    import flb_native as nat
    return nat.lib.flb_layer_norm_bwd(x, ldx, codes, exps, mean, rstd, w, wdt, dy, dx, dw, db, G, R, D, dt, ws, n, None)


def test_norm_arguments():
    """Every refusal comes before any device work: the pointers here are not memory."""
    import flb_native as nat
    assert norm_fwd(dt=7) == FLB_DTYPE and norm_fwd(w=16, wdt=F16) == FLB_DTYPE
    assert norm_fwd(D=0) == FLB_SHAPE and norm_fwd(R=-1) == FLB_SHAPE and norm_fwd(G=-1) == FLB_SHAPE and norm_fwd(ldx=-8) == FLB_SHAPE
    assert norm_fwd(D=32769) == FLB_UNSUPPORTED and norm_fwd(G=65536) == FLB_UNSUPPORTED
    assert norm_fwd(R=2 ** 31) == FLB_SHAPE and norm_fwd(G=65535, R=2 ** 16) == FLB_SHAPE
    assert norm_fwd(x=None) == FLB_SHAPE and norm_fwd(y=None) == FLB_SHAPE
    assert norm_fwd(codes=16) == FLB_SHAPE and norm_fwd(exps=16) == FLB_SHAPE and norm_fwd(codes=8, exps=8) == FLB_ALIGN
    assert norm_fwd(x=1) == FLB_ALIGN and norm_fwd(w=2) == FLB_ALIGN and norm_fwd(rstd=2) == FLB_ALIGN
    assert norm_fwd(R=0, x=None, y=None) == 0 and norm_fwd(G=0, x=None, y=None) == 0
    assert norm_bwd(D=16385) == FLB_UNSUPPORTED and norm_bwd(dy=None) == FLB_SHAPE and norm_bwd(mean=None) == FLB_SHAPE
    assert norm_bwd(rstd=None) == FLB_SHAPE and norm_bwd(dw=16) == FLB_SHAPE and norm_bwd(dx=3) == FLB_ALIGN
    assert norm_bwd(x=None, codes=16) == FLB_SHAPE
    need = nat.lib.flb_layer_norm_bwd_workspace_bytes(1, 4096, 768)
    assert need > 0 and nat.lib.flb_layer_norm_bwd_workspace_bytes(1, 4, 768) == 0
    assert norm_bwd(dw=16, db=16, R=4096, D=768, ldx=768) == FLB_WORKSPACE
    assert norm_bwd(dw=16, db=16, R=4096, D=768, ldx=768, ws=16, n=need - 1) == FLB_WORKSPACE
    assert norm_bwd(dw=16, db=16, R=4096, D=768, ldx=768, ws=24, n=need) == FLB_ALIGN
    assert b"workspace" in nat.lib.flb_last_error()


def test_kept_arguments():
    import flb_native as nat
    L = nat.lib
    assert L.flb_code_pitch(1) == 16 and L.flb_code_pitch(16) == 16 and L.flb_code_pitch(17) == 32 and L.flb_code_pitch(0) == 0
    assert L.flb_kept_blocks(128) == 1 and L.flb_kept_blocks(129) == 2
    assert L.flb_pack8(16, 16, 16, 1, 8, 5, None) == FLB_DTYPE and L.flb_pack8(16, 16, 16, -1, 8, F32, None) == FLB_SHAPE
    assert L.flb_pack8(16, 16, 16, 1, 0, F32, None) == FLB_SHAPE and L.flb_pack8(None, 16, 16, 1, 8, F32, None) == FLB_SHAPE
    assert L.flb_pack8(16, 16, None, 1, 8, F32, None) == FLB_SHAPE and L.flb_pack8(16, 24, 16, 1, 8, F32, None) == FLB_ALIGN
    assert L.flb_pack8(18, 16, 16, 1, 8, F32, None) == FLB_ALIGN and L.flb_pack8(16, 16, 16, 2 ** 62, 8, F32, None) == FLB_SHAPE
    assert L.flb_unpack8(16, 16, None, 1, 8, F32, None) == FLB_SHAPE and L.flb_unpack8(16, 16, 18, 1, 8, F32, None) == FLB_ALIGN
    assert L.flb_pack8(None, None, None, 0, 8, F32, None) == 0 and L.flb_unpack8(None, None, None, 0, 8, F32, None) == 0
    assert L.flb_gate_fwd(16, 16, 16, 16, 16, None, None, 1, 8, F32, None) == FLB_SHAPE
    assert L.flb_gate_fwd(16, None, 16, None, None, None, None, 1, 8, F32, None) == FLB_SHAPE
    assert L.flb_gate_bwd(None, None, None, None, None, None, 16, 16, 16, 1, 8, F32, None) == FLB_SHAPE
    assert L.flb_gate_bwd(16, 16, None, None, None, None, 16, 16, 17, 1, 8, F16, None) == FLB_ALIGN
    assert L.flb_gate_bwd(None, None, None, None, None, None, None, None, None, 0, 8, F16, None) == 0


def int8(x=16, ldx=64, xc=None, ldc=0, xs=None, wc=16, ldw=64, ws=16, bias=None, bdt=F32, out=16, M=4, N=8, K=64, dt=BF16, work=256,
         n=1 << 30):
    import flb_native as nat
    return nat.lib.flb_int8_linear(x, ldx, xc, ldc, xs, wc, ldw, ws, bias, bdt, out, M, N, K, dt, work, n, 0, None)


def test_int8_arguments():
    """Every refusal comes before any device work."""
    import flb_native as nat
    L = nat.lib
    assert int8(dt=9) == FLB_DTYPE and int8(bias=16, bdt=F16) == FLB_DTYPE
    assert int8(M=-1) == FLB_SHAPE and int8(N=-1) == FLB_SHAPE and int8(K=0) == FLB_SHAPE and int8(K=32769) == FLB_UNSUPPORTED
    assert int8(M=2 ** 31) == FLB_SHAPE and int8(M=2 ** 30, N=2 ** 30) == FLB_SHAPE
    assert int8(x=None) == FLB_SHAPE and int8(xc=16, xs=16, ldc=64) == FLB_SHAPE and int8(x=None, xc=16) == FLB_SHAPE
    assert int8(wc=None) == FLB_SHAPE and int8(ws=None) == FLB_SHAPE and int8(out=None) == FLB_SHAPE
    assert int8(ldx=-1) == FLB_SHAPE and int8(ldw=48) == FLB_SHAPE and int8(x=None, xc=16, xs=16, ldc=48) == FLB_SHAPE
    assert int8(ldw=72) == FLB_ALIGN and int8(wc=8) == FLB_ALIGN and int8(x=None, xc=24, xs=16, ldc=64) == FLB_ALIGN
    assert int8(x=17) == FLB_ALIGN and int8(out=17) == FLB_ALIGN and int8(ws=18) == FLB_ALIGN
    assert int8(work=None) == FLB_WORKSPACE and int8(n=16) == FLB_WORKSPACE and int8(work=128) == FLB_ALIGN
    assert int8(M=0, x=None, out=None) == 0 and int8(N=0, wc=None, ws=None) == 0
    assert L.flb_int8_linear_workspace_bytes(400, 8, 64, 0) > L.flb_int8_linear_workspace_bytes(400, 8, 64, 1) > 0
    assert L.flb_int8_linear_workspace_bytes(4, 8, 64, 0) > 0
    assert L.flb_int8_linear_workspace_bytes(0, 8, 64, 0) == 0 and L.flb_int8_linear_workspace_bytes(4, 8, 0, 0) == 0
    assert L.flb_int8_rows(16, 8, 16, 16, 2, 8, 5, None) == FLB_DTYPE and L.flb_int8_rows(16, 8, 24, 16, 2, 8, F32, None) == FLB_ALIGN
    assert L.flb_int8_rows(None, 8, 16, 16, 2, 8, F32, None) == FLB_SHAPE and L.flb_int8_rows(None, 8, None, None, 0, 8, F32, None) == 0
    assert L.flb_layer_norm_int8(16, 8, 16, None, F16, 16, 16, 1, 2, 8, BF16, 1e-5, None) == FLB_DTYPE
    assert L.flb_layer_norm_int8(16, 8, None, None, F32, None, 16, 1, 2, 8, BF16, 1e-5, None) == FLB_SHAPE


def test_kept_training_arguments():
    import flb_native as nat
    L = nat.lib
    assert L.flb_block_grid_saved8_bytes(0, 4, 2, 64) == 0
    b16, b8 = L.flb_block_grid_saved_bytes(4, 6, 3, 128), L.flb_block_grid_saved8_bytes(4, 6, 3, 128)
    assert b8 <= 4 * 6 * 3 * 18 * 129 + 256 and b16 == 4 * 6 * 3 * 36 * 128 * 2
    assert L.flb_block_grid_fwd_save8(None, 16, 16, 4, 6, 3, 64, 8, 1e-5, 16, 1 << 30, 16, 1 << 30, None) == FLB_SHAPE
    assert L.flb_block_grid_bwd_saved8(None, 16, 16, None, None, None, None, 16, 16, 4, 6, 3, 64, 8, 1e-5, 16, 1 << 30, 16, 1 << 30,
                                       None) == FLB_SHAPE


def test_rows_of_views():
    """Which views the kernels take as they are, and which are copied."""
    from flb_ops import rows_of as as_rows
    t = torch.arange(5 * 8 * 12.).reshape(5, 8, 12)
    for v, pitch, same in ((t, 12, True), (t[:, :, 2:6], 12, True), (t[:, ::2, :4], 24, True), (t[:, :3], None, False),
                           (t.transpose(0, 1), None, False), (t[:1, :1, :5], 5, None), (t[..., ::2], 6, False), (t[2:3, :, 1:4], 12, True)):
        x, ld = as_rows(v)
        rows = v.numel() // v.shape[-1]
        flat = torch.as_strided(x, (rows, v.shape[-1]), (ld, 1), x.storage_offset())
        assert torch.equal(flat, v.reshape(rows, -1))
        if pitch is not None:
            assert ld == pitch
        if same is not None:
            assert (x.data_ptr() == v.data_ptr()) == same


def test_kept_oracle():
    """The oracle's own rule: units are powers of two, codes fill 64 to 127, errors are at most half a unit."""
    from oracle import rows as orc
    x = torch.randn(9, 300, dtype=torch.float64) * torch.exp(3 * torch.randn(9, 1, dtype=torch.float64))
    v, unit, _ = orc.kept(x)
    assert torch.equal(torch.frexp(unit)[0], torch.full_like(unit, 0.5)) and ((v - x).abs() <= unit / 2).all()
    top = (v / unit).abs()[:, :128].amax(-1)
    assert (top >= 64).all() and (top <= 127).all()
