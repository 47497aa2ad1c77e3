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


def _cast64(x, block_rows):
    """Values of the codes, scales and each quotient's relative distance to the nearest tie, in 64 bits."""
    M, K = x.shape
    mb, kb = -(-M // block_rows), -(-K // 128)
    pad = torch.nn.functional.pad(x.double(), (0, kb * 128 - K, 0, mb * block_rows - M)).view(mb, block_rows, kb, 128)
    amax = pad.abs().amax((1, 3)).clamp(min=1e-12)
    q = (448.0 * pad / amax[:, None, :, None]).view(mb * block_rows, kb * 128)[:M, :K]
    a = q.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    v = torch.minimum(torch.round(a / step) * step, torch.tensor(448.0, device=x.device, dtype=torch.float64))
    return torch.sign(q) * v, amax / 448.0, ((a / step) % 1 - 0.5).abs() * step / a.clamp(min=1e-300)


# (far more blocks than the launch's half-warps, 16 x 5 per SM, so that every one goes on from row to row; the number
# of blocks per row divides that number, or leaves a remainder)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K,block_rows", [(65536, 64, 1), (30000, 129, 1), (12001, 512, 1), (8000, 1171, 1), (8001, 1176, 1), (4100, 3200, 1),
                                            (3001, 8192, 1), (700, 30000, 1), (5120, 1280, 128), (1000, 4100, 128)])
def test_casts_of_many_blocks_match_the_formula(M, K, block_rows, dtype):
    """Tolerances as beside the small cases (test_fp8_block_gpu.py): none for bf16, a code next to a tie for fp32."""
    from vitfp4.nvfp4 import quantize_to_fp8_block
    if block_rows == 1:
        assert M * -(-K // 128) > 3 * 80 * torch.cuda.get_device_properties(0).multi_processor_count
    x = torch.randn(M, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(K))
    x[:, :: max(1, K // 3)] *= 20
    x = (x * torch.arange(1, M + 1, device="cuda")[:, None]).to(dtype)      # every row's scales are its own
    codes, scale = quantize_to_fp8_block(x, block_rows)
    v, s, tie = _cast64(x, block_rows)
    assert ((scale.double() - s).abs() <= s * (2.0 ** -24 * 1.001)).all()
    off = codes.double() != v
    assert not (off & (tie > (0.0 if dtype == torch.bfloat16 else 2.0 ** -23))).any(), int(off.sum())


@pytest.mark.parametrize("M,K,N", [(4000, 1176, 300), (2500, 1171, 1001)])
def test_a_linear_layer_of_many_rows_is_its_cast_and_product(M, K, N):
    from vitfp4.nvfp4 import fp8_block_gemm, fp8_block_linear, quantize_to_fp8_block
    x = torch.randn(M, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(M)).bfloat16()
    w, ws = quantize_to_fp8_block(torch.randn(N, K, device="cuda"), 128)
    a, sa = quantize_to_fp8_block(x)
    assert torch.equal(fp8_block_linear(x, w, ws), fp8_block_gemm(a, sa, w, ws))
