"""FP8 block operands of other numbers of dimensions, and casts that go on over many blocks."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("K", [256, 200])
def test_the_product_takes_what_the_cast_and_the_norm_return(K):
    from vitfp4.nvfp4 import fp8_block_gemm, gated_residual_norm, quantize_to_fp8_block
    x, y = torch.randn(2, 3, 5, 7, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(K)).bfloat16()
    w, ws = quantize_to_fp8_block(torch.randn(140, K, device="cuda"), 128)
    bias = torch.randn(140, device="cuda")
    for t in (x, x[0], x[0, 0], x[0, 0, 0], x[:, :0]):
        a, sa = quantize_to_fp8_block(t)
        for dt in (torch.bfloat16, torch.float32):
            want = fp8_block_gemm(a.reshape(-1, K), sa.reshape(-1, sa.shape[-1]), w, ws, bias=bias, out_dtype=dt)
            got = fp8_block_gemm(a, sa, w, ws, bias=bias, out_dtype=dt)
            assert got.shape == (*t.shape[:-1], 140) and got.dtype == dt and torch.equal(got.reshape(-1, 140), want)
    _, (h, sh) = gated_residual_norm(x, y, out_dtype=F8)
    got = fp8_block_gemm(h, sh, w, ws)
    assert got.shape == (3, 5, 7, 140)
    assert torch.equal(got.view(-1, 140), fp8_block_gemm(h.reshape(-1, K), sh.reshape(-1, sh.shape[-1]), w, ws))
