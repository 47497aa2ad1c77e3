"""gated_residual_norm with more rows than the machine takes at once, so that every warp and CTA goes on to further rows,
in each of its forms, against the formula in 64 bits.  Tolerances: as derived beside the small cases
(test_gated_norm_gpu.py); without y, x' is x and has no error of its own."""
import pytest
import torch
from test_gated_norm_gpu import DT, EPS, _c, _case, _near, _norm64, _want

pytestmark = pytest.mark.gpu

FORMS = ["both", "pre", "post", "no y"]


def _check(form, x, y, gate, w2, b2, w1, b1, norm):
    from vitfp4.nvfp4 import gated_residual_norm
    post = dict(post_weight=w2, post_bias=b2) if form in ("both", "post") else dict(post_norm=False)
    pre = dict(pre_weight=w1, pre_bias=b1) if form != "post" else dict(pre_norm=False)
    if form == "no y":
        new, h = gated_residual_norm(x, None, norm=norm, eps=EPS, **pre)
        assert new is x
        want = x.double()
        hw = _norm64(want, norm, w1, b1)
        rms = torch.sqrt((_c(want, norm) ** 2).mean(1, keepdim=True) + EPS)
        B = hw.abs().amax(1, keepdim=True) + 1
        e2 = 1.5 * 2.0 ** -24 * (100 * (B + want.abs().amax(1, keepdim=True) / rms) + 10)
    else:
        new, h = gated_residual_norm(x, y, gate=gate, residual_scale=0.7, norm=norm, eps=EPS, **post, **pre)
        if form == "pre":
            w2 = b2 = None
        want, hw, e1, e2 = _want(x, y, gate, w2, b2, w1, b1, norm, 0.7, post=form != "pre")
        _near(new, want, e1, "x'")
    if form == "post":
        assert h is None
    else:
        _near(h, hw, e2, "h")


# a CTA per row: 16 CTAs per SM are launched
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("K", [1536, 2048, 3001, 5120])
def test_a_cta_takes_several_rows(K, norm, form):
    M = 5000
    assert M > 2 * 16 * torch.cuda.get_device_properties(0).multi_processor_count
    _check(form, *_case(M, K, "bf16", 0 if form == "no y" else 8, True, norm, seed=K), norm)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("K", [2048, 4096])
def test_a_cta_takes_several_fp32_rows(K, form):
    _check(form, *_case(5001, K, "f32", 0, False, "rms", seed=K), "rms")


# a warp per row: 8 rows per CTA, up to three CTAs per SM
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("K", [200, 320, 512, 768, 1001, 1024, 1280])
@pytest.mark.parametrize("groups,norm,dtype", [(1, "layer", "bf16"), (25, "rms", "bf16"), (72, "layer", "f32")])
def test_a_warp_takes_several_rows(groups, norm, dtype, K, form):
    M = 7200
    assert M > 2 * 3 * 8 * torch.cuda.get_device_properties(0).multi_processor_count
    _check(form, *_case(M, K, dtype, 0 if form == "no y" else groups, True, norm, seed=K + groups), norm)


@pytest.mark.parametrize("M,K", [(7200, 1024), (7201, 1279), (5000, 5120)])
def test_fp8_output_of_many_rows(M, K):
    from vitfp4.nvfp4 import dequantize_fp8_block, gated_residual_norm
    x, y, gate, w2, b2, w1, b1 = _case(M, K, "bf16", 1, True, "rms", seed=K)
    kw = dict(gate=gate, residual_scale=0.5, norm="rms", post_weight=w2, pre_weight=w1, eps=EPS)
    new, (codes, scale) = gated_residual_norm(x, y, out_dtype=torch.float8_e4m3fn, **kw)
    assert torch.equal(new, gated_residual_norm(x, y, **kw)[0])
    _, hw, _, e2 = _want(x, y, gate, w2, b2, w1, b1, "rms", 0.5)
    amax = torch.nn.functional.pad(hw, (0, -K % 128)).view(M, -1, 128).abs().amax(2)
    assert ((scale.double() * 448 - amax).abs() <= e2 + amax * 2.0 ** -23).all()
    # half a step of E4M3: 2^-4 of the value, or half of the smallest step (2^-10) of the block's scale
    step = torch.maximum(hw.abs() * 2.0 ** -4, (amax / 448 * 2.0 ** -10).repeat_interleave(128, 1)[:, :K])
    d = dequantize_fp8_block(codes, scale).double()
    assert ((d - hw).abs() <= step * (1 + 2.0 ** -20) + 2 * e2).all()
    assert DT["bf16"] == new.dtype


@pytest.mark.parametrize("size", [1.0, 5e37, 2e-13, float("inf")])
@pytest.mark.parametrize("M,K", [(5, 100), (300, 1024), (3000, 1280), (33, 2048), (9, 5120), (7, 3001)])
def test_fp8_output_is_bit_for_bit_the_cast(M, K, size):
    """fp32 rows come out unrounded, so casting them has to give the codes and scales that the fused output holds: at a
    usual size, above 2^126 (where an approximate quotient 448 / amax would be 0), at a block maximum near the least
    one, and with an infinite value in every row."""
    from vitfp4.nvfp4 import gated_residual_norm, quantize_to_fp8_block
    x, y, gate, w2, _, w1, _ = _case(M, K, "f32", 1, True, "rms", seed=K)
    if size == float("inf"):
        w1[K // 3] = size
    else:
        w1 = w1 * size
    kw = dict(gate=gate, residual_scale=0.5, norm="rms", post_weight=w2, pre_weight=w1, eps=EPS)
    _, h = gated_residual_norm(x, y, **kw)
    assert h.abs().amax() > 2.0 ** 126 if size > 1 else h.isfinite().all()
    _, (codes, scale) = gated_residual_norm(x, y, out_dtype=torch.float8_e4m3fn, **kw)
    want, ws = quantize_to_fp8_block(h)
    assert torch.equal(scale, ws)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
