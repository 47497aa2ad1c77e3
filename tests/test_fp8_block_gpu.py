"""FP8 block format on the GPU: the cast against the formula in 64 bits, the product against a sum in 64 bits.

Tolerances.  Cast of bf16: none -- 448 x / amax is a quotient of integers below 2^12 and 2^8, so unless it lies
exactly between two codes it is further from such a point than fp32 rounding moves it.  Cast of fp32: the code may
differ where the quotient lies within 2^-23 (relative) of a point between two codes.  Scales: one fp32 rounding.
Product: the products of two codes are exact in fp32; each of the K additions inside blocks and of the ceil(K/128)
block sums (scaled by a product of two scales, three more roundings) may lose one unit (2^-23: the tensor core
truncates) of at most the sum of magnitudes: |err| <= (K + 4 ceil(K/128)) 2^-23 sum |a b| s, plus the bias add and the
rounding to the output type, half a step each.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _e4m3(q: np.ndarray):
    """Nearest E4M3 value (ties to even) of float64 q, saturating; and the distance to the nearest tie, relative."""
    a = np.abs(q)
    step = np.exp2(np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    v = np.minimum(np.round(a / step) * step, 448.0)
    frac = a / step - np.floor(a / step)
    return np.sign(q) * v, np.abs(frac - 0.5) * step / np.maximum(a, 1e-300)


def _cast64(x: np.ndarray, block_rows: int):
    M, K = x.shape
    mb, kb = -(-M // block_rows), -(-K // 128)
    amax = np.full((mb, kb), 1e-12)
    for i in range(mb):
        for g in range(kb):
            amax[i, g] = max(np.abs(x[i * block_rows:(i + 1) * block_rows, g * 128:(g + 1) * 128]).max(), 1e-12)
    full = np.repeat(np.repeat(amax, block_rows, 0)[:M], 128, 1)[:, :K]
    v, tie = _e4m3(448.0 * x / full)
    return v, amax / 448.0, tie


def _x(M, K, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, device="cuda", generator=g) * scale
    x[:, :: max(1, K // 3)] *= 20
    return x.to(DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 7), (2, 120), (5, 129), (129, 255), (257, 1024), (64, 1176),
                                 (300, 1000), (33, 8192)])
def test_cast_matches_formula(M, K, block_rows, dtype):
    from vitfp4.nvfp4 import quantize_to_fp8_block
    x = _x(M, K, dtype, seed=M * 7 + K)
    codes, scale = quantize_to_fp8_block(x, block_rows)
    assert codes.shape == (M, K) and codes.dtype == torch.float8_e4m3fn
    v, s, tie = _cast64(x.double().cpu().numpy(), block_rows)
    np.testing.assert_allclose(scale.double().cpu().numpy(), s, rtol=2 ** -24 * 1.001)
    off = codes.double().cpu().numpy() != v
    assert not (off & (tie > (0.0 if dtype == "bf16" else 2.0 ** -23))).any(), off.sum()


@pytest.mark.parametrize("scale", [1e-30, 1e-15, 1e30, 1e37])
def test_cast_extreme_magnitudes(scale):
    from vitfp4.nvfp4 import quantize_to_fp8_block
    x = (torch.randn(8, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * scale).bfloat16()
    codes, s = quantize_to_fp8_block(x)
    v, s64, _ = _cast64(x.double().cpu().numpy(), 1)
    assert np.array_equal(codes.double().cpu().numpy(), v)
    np.testing.assert_allclose(s.double().cpu().numpy(), s64, rtol=2 ** -24 * 1.001)


def test_cast_zero_nan_and_infinity():
    from vitfp4.nvfp4 import dequantize_fp8_block, quantize_to_fp8_block
    x = torch.ones(4, 256, device="cuda", dtype=torch.bfloat16)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 200] = float("-inf")
    codes, scale = quantize_to_fp8_block(x)
    d = dequantize_fp8_block(codes, scale)
    assert (d[0] == 0).all() and (scale[0] > 0).all()
    assert d[1, :128].isnan().all() and (d[1, 128:] == 1).all()
    c2 = codes.float()[2]
    assert (d[2, :128] == 1).all() and c2[200].isnan() and (c2[128:200] == 0).all() and (c2[201:] == 0).all()
    assert (d[3] == 1).all()


def test_cast_strided_unaligned_and_batched():
    from vitfp4.nvfp4 import quantize_to_fp8_block
    big = _x(40, 600, "bf16", seed=5)
    for view in (big[:, 3:300], big[:, 8:264], big[::2, :256], big.t()[:, :37], big[:1, 1:130]):
        codes, scale = quantize_to_fp8_block(view)
        want, ws = quantize_to_fp8_block(view.contiguous().clone())
        assert torch.equal(codes.float(), want.float()) and torch.equal(scale, ws)
    c3, s3 = quantize_to_fp8_block(big.view(4, 10, 600))
    c2, s2 = quantize_to_fp8_block(big)
    assert c3.shape == (4, 10, 600) and torch.equal(c3.view(40, 600).float(), c2.float())
    assert torch.equal(s3.reshape(40, -1), s2)
    empty, es = quantize_to_fp8_block(big[:0])
    assert empty.shape == (0, 600) and es.shape == (0, 5)


def _operands(M, N, K, seed=0):
    from vitfp4.nvfp4 import quantize_to_fp8_block
    a = quantize_to_fp8_block(_x(M, K, "bf16", seed))
    w = torch.randn(N, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 1)) * 0.05
    return a, quantize_to_fp8_block(w, 128)


def _product64(a, sa, b, sb):
    """(sum, sum of magnitudes) in 64 bits."""
    K, N = a.shape[1], b.shape[0]
    A = a.double() * sa.double().repeat_interleave(128, 1)[:, :K]
    B = b.double() * sb.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return A @ B.t(), A.abs() @ B.abs().t()


def _check(y, want, mag, K, bias=None, wide=None):
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    eps = torch.finfo(y.dtype).eps / 2
    tol = (K + 4 * -(-K // 128)) * 2.0 ** -23 * mag + want.abs() * (eps + 2.0 ** -24) + 1e-30
    bad = (y.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((y.double() - want).abs() / tol).max()))


SIZES = [(1, 1, 1), (1, 8, 16), (2, 100, 130), (5, 128, 128), (16, 129, 300), (17, 257, 1024), (33, 64, 2048), (64, 1000, 520),
         (65, 128, 256), (128, 1, 100), (129, 255, 640), (257, 1000, 1176), (300, 2049, 64), (1000, 520, 2000),
         (2560, 2048, 300), (2500, 2100, 140)]


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_matches_sum_in_64_bits(M, N, K, out):
    from vitfp4 import _lib
    from vitfp4.nvfp4 import fp8_block_gemm
    (a, sa), (b, sb) = _operands(M, N, K, seed=M + N + K)
    bias = torch.randn(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)).to(DT[out])
    want, mag = _product64(a, sa, b, sb)
    y = fp8_block_gemm(a, sa, b, sb, out_dtype=DT[out])
    assert y.dtype == DT[out] and y.shape == (M, N)
    _check(y, want, mag, K)
    yb = fp8_block_gemm(a, sa, b, sb, bias=bias, out_dtype=DT[out])
    _check(yb, want, mag, K, bias)
    assert torch.equal(yb, fp8_block_gemm(a, sa, b, sb, bias=bias, out_dtype=DT[out]))   # no timing in the result
    assert _lib.device_error() == 0


@pytest.mark.parametrize("M", [3, 40, 200])
def test_product_strides_layouts_and_bytes_past_k(M):
    from vitfp4.nvfp4 import fp8_block_gemm
    (a, sa), (b, sb) = _operands(M, 200, 200, seed=M)
    want = fp8_block_gemm(a, sa, b, sb)
    nan = torch.full((M, 256), float("nan"), device="cuda").to(torch.float8_e4m3fn)
    nan[:, :200] = a                                    # the row's bytes past K are NaN codes
    wnan = torch.full((200, 320), float("nan"), device="cuda").to(torch.float8_e4m3fn)
    wnan[:, 16:216] = b
    assert torch.equal(fp8_block_gemm(nan[:, :200], sa.contiguous(), wnan[:, 16:216], sb.t().contiguous().t()), want)
    odd = torch.empty(M, 203, device="cuda").to(torch.float8_e4m3fn)
    odd[:, 1:201] = a                                   # rows off the 16-byte boundaries are copied
    assert torch.equal(fp8_block_gemm(odd[:, 1:201], sa, b, sb), want)
    tight = a.contiguous()                              # rows of exactly K bytes
    assert torch.equal(fp8_block_gemm(tight, sa, b, sb), want)


@pytest.mark.parametrize("M", [4, 50, 150])
def test_product_nan_row_stays_in_its_row(M):
    from vitfp4.nvfp4 import fp8_block_linear, quantize_to_fp8_block
    x = _x(M, 256, "bf16", seed=2)
    w = quantize_to_fp8_block(torch.randn(130, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)), 128)
    clean = fp8_block_linear(x, *w)
    x[2, 7] = float("nan")
    y = fp8_block_linear(x, *w)
    assert y[2].isnan().all()
    keep = torch.arange(M, device="cuda") != 2
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape,N,K", [((1,), 300, 1024), ((2, 1), 1000, 1000), ((3,), 77, 515), ((4,), 4096, 128), ((7,), 130, 260),
                                       ((2, 3, 11), 256, 384), ((257,), 512, 768), ((0,), 64, 64)])
def test_linear_is_cast_then_product(shape, N, K, dtype):
    from vitfp4.nvfp4 import fp8_block_linear, quantize_to_fp8_block
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(*shape, K, device="cuda", generator=g).to(DT[dtype])
    w, ws = quantize_to_fp8_block(torch.randn(N, K, device="cuda", generator=g) * 0.05, 128)
    bias = torch.randn(N, device="cuda", generator=g).bfloat16()
    y = fp8_block_linear(x, w, ws, bias=bias)
    assert y.shape == (*shape, N) and y.dtype == x.dtype
    if x.numel():
        codes, scale = quantize_to_fp8_block(x.reshape(-1, K))
        want, mag = _product64(codes, scale, w, ws)
        _check(y.reshape(-1, N), want, mag, K, bias)


# one and two rows in one launch: several passes over the weight rows, up to four chunks of columns; narrow tiles with
# more tiles than CTAs and an odd number of K blocks, and shared by clusters of each size; two waves of 128 x 128 tiles
@pytest.mark.parametrize("M,N,K", [(1, 9001, 500), (2, 8192, 512), (1, 700, 2047), (1, 701, 2049), (2, 5000, 1024), (16, 38100, 384),
                                   (17, 38100, 300), (40, 19300, 384), (16, 1000, 1300), (31, 4900, 2600), (64, 1000, 1300),
                                   (50, 5000, 2700), (100, 2200, 1700), (2050, 1280, 260)])
def test_linear_at_the_edges_of_its_variants(M, N, K):
    from vitfp4.nvfp4 import fp8_block_linear, quantize_to_fp8_block
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    w, ws = quantize_to_fp8_block(torch.randn(N, K, device="cuda", generator=g) * 0.05, 128)
    bias = torch.randn(N, device="cuda", generator=g).bfloat16()
    codes, scale = quantize_to_fp8_block(x)
    want, mag = _product64(codes, scale, w, ws)
    y = fp8_block_linear(x, w, ws, bias=bias)
    _check(y, want, mag, K, bias)
    assert torch.equal(y, fp8_block_linear(x, w, ws, bias=bias))   # no order of additions depends on timing


def test_linear_captured_replayed_and_on_another_stream():
    from vitfp4.nvfp4 import fp8_block_linear, quantize_to_fp8_block
    g = torch.Generator(device="cuda").manual_seed(4)
    w, ws = quantize_to_fp8_block(torch.randn(512, 640, device="cuda", generator=g), 128)
    for M in (1, 30, 200):
        xs = [torch.randn(M, 640, device="cuda", generator=g).bfloat16() for _ in range(3)]
        want = [fp8_block_linear(x, w, ws) for x in xs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [fp8_block_linear(x, w, ws) for x in xs]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        buf = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp8_block_linear(buf, w, ws)
        for x, r in zip(xs, want):
            buf.copy_(x)
            graph.replay()
            assert torch.equal(y, r)
