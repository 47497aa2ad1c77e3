"""gated_residual_norm on the GPU against the formula in 64 bits.

Tolerances.  A sum of K fp32 terms over a row's threads is off by at most (log2 of the tree and the serial part,
under 40 additions) 40 * 2^-24 of the sum of magnitudes, so a mean is off by at most 40 * 2^-24 * max|v| and a variance
by as much of itself plus twice the mean's share; rsqrt, four products and two additions follow.  With values
of a row bounded by A (after centring, in units of its rms) a normalised value is off by at most u = 2^-24 * (40 * A +
40 * |z| + 10 * |z| + 4): e = 2^-24 * (100 * A + 10) covers |z| <= A.  The first norm's error enters x' times |rs * gate * w|,
and the second norm divides by the rms of x'.  Rounding to the output type adds half a step of the value.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def _norm64(v, kind, w, b):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
    v = v if w is None else v * w.double()
    return v if b is None else v + b.double()


def _case(M, K, dtype, groups, affine, norm, seed=0, pdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    dt, pt = DT[dtype], DT[pdtype or dtype]
    x, y = (r(M, K) + 0.5).to(dt), (2 * r(M, K) - 0.3).to(dt)
    gate = None if groups == 0 else (r(K) if groups == 1 else r(groups, K)).to(pt)
    w2, w1 = ((1 + 0.1 * r(K)).to(pt), (1 + 0.1 * r(K)).to(pt)) if affine else (None, None)
    b2, b1 = ((0.1 * r(K)).to(pt), (0.1 * r(K)).to(pt)) if affine and norm == "layer" else (None, None)
    return x, y, gate, w2, b2, w1, b1


def _want(x, y, gate, w2, b2, w1, b1, norm, rs, post=True):
    """x', h and the bounds on their errors before rounding."""
    M = x.shape[0]
    z = _norm64(y.double(), norm, w2, b2) if post else y.double()
    gg = torch.ones_like(z) if gate is None else gate.double().view(-1, x.shape[1]).repeat_interleave(
        M // (1 if gate.dim() == 1 else gate.shape[0]), 0)
    new = x.double() + rs * gg * z
    A = z.abs().amax(1, keepdim=True) + 1
    e1 = 2.0 ** -24 * ((100 * A + 10) * (rs * gg).abs() * (1.5 if post else 0) + 4 * new.abs() + 4 * x.double().abs())
    h = _norm64(new, norm, w1, b1)
    rms = torch.sqrt((_c(new, norm) ** 2).mean(1, keepdim=True) + EPS)
    B = h.abs().amax(1, keepdim=True) + 1
    e2 = 1.5 * e1.amax(1, keepdim=True) * (1 + B) * 2 / rms + 1.5 * 2.0 ** -24 * (100 * (B + new.abs().amax(1, keepdim=True) / rms) + 10)
    return new, h, e1, e2


def _c(v, norm):
    return v - v.mean(1, keepdim=True) if norm == "layer" else v


def _near(got, want, err, what):
    tol = err + want.abs() * (torch.finfo(got.dtype).eps / 2 * 1.001) + 1e-30
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


SIZES = [(1, 1), (1, 8), (3, 130), (5, 255), (17, 256), (9, 504), (257, 1024), (6, 1000), (4, 1025), (7, 2048), (3, 3001), (2, 4096),
         (5, 5120), (2, 8191), (2, 16384)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("M,K", SIZES)
def test_matches_formula(M, K, norm, dtype):
    from vitfp4.nvfp4 import gated_residual_norm
    if K == 1 and norm == "layer":
        pytest.skip("one column has no variance: 0 / sqrt(eps), tested below")
    x, y, gate, w2, b2, w1, b1 = _case(M, K, dtype, 1, True, norm, seed=M + K)
    new, h = gated_residual_norm(x, y, gate=gate, residual_scale=0.7, norm=norm, post_weight=w2, post_bias=b2,
                                 pre_weight=w1, pre_bias=b1, eps=EPS)
    want, hw, e1, e2 = _want(x, y, gate, w2, b2, w1, b1, norm, 0.7)
    assert new.dtype == x.dtype and h.dtype == x.dtype
    _near(new, want, e1, "x'")
    _near(h, hw, e2, "h")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("groups", [0, 2, 3, 12])
@pytest.mark.parametrize("affine", [False, True])
def test_gates_per_group_and_missing_parts(groups, affine, dtype):
    from vitfp4.nvfp4 import gated_residual_norm
    M, K = 12, 320
    x, y, gate, w2, b2, w1, b1 = _case(M, K, dtype, groups, affine, "layer", seed=groups)
    kw = dict(gate=gate, residual_scale=-1.25, eps=EPS)
    new, h = gated_residual_norm(x, y, post_weight=w2, post_bias=b2, pre_weight=w1, pre_bias=b1, **kw)
    want, hw, e1, e2 = _want(x, y, gate, w2, b2, w1, b1, "layer", -1.25)
    _near(new, want, e1 * 2, "x'")
    _near(h, hw, e2 * 2, "h")
    new, h = gated_residual_norm(x, y, post_norm=False, pre_weight=w1, pre_bias=b1, **kw)
    want, hw, e1, e2 = _want(x, y, gate, None, None, w1, b1, "layer", -1.25, post=False)
    _near(new, want, e1, "x' without post-norm")
    _near(h, hw, e2, "h without post-norm")
    new2, none = gated_residual_norm(x, y, post_norm=False, pre_norm=False, **kw)
    assert none is None and torch.equal(new2, new)
    same, h = gated_residual_norm(x, None, pre_weight=w1, pre_bias=b1, eps=EPS)
    assert same is x
    _near(h, _norm64(x.double(), "layer", w1, b1), 2.0 ** -24 * 2000, "pre-norm alone")


def test_parameters_of_the_other_type():
    from vitfp4.nvfp4 import gated_residual_norm
    for dtype, pd in (("bf16", "f32"), ("f32", "bf16")):
        x, y, gate, w2, b2, w1, b1 = _case(20, 264, dtype, 4, True, "layer", seed=1, pdtype=pd)
        kw = dict(residual_scale=0.5, eps=EPS)
        new, h = gated_residual_norm(x, y, gate=gate, post_weight=w2, post_bias=b2, pre_weight=w1, pre_bias=b1, **kw)
        want, hw, e1, e2 = _want(x, y, gate, w2, b2, w1, b1, "layer", 0.5)
        _near(new, want, e1, "x'")
        _near(h, hw, e2, "h")
        mixed, hm = gated_residual_norm(x, y, gate=gate, post_weight=w2.float(), post_bias=b2, pre_weight=w1, pre_bias=b1, **kw)
        if pd == "bf16":   # mixed types are taken to fp32, exactly
            assert torch.equal(mixed, new) and torch.equal(hm, h)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("M,K", [(1, 128), (5, 100), (33, 1024), (9, 1176), (3, 5120), (2, 3001)])
def test_fp8_output_is_the_cast_of_the_unrounded_norm(M, K, dtype):
    from vitfp4.nvfp4 import dequantize_fp8_block, gated_residual_norm
    x, y, gate, w2, b2, w1, b1 = _case(M, K, dtype, 1, True, "rms", seed=K)
    kw = dict(gate=gate, residual_scale=0.5, norm="rms", post_weight=w2, pre_weight=w1, eps=EPS)
    new, (codes, scale) = gated_residual_norm(x, y, out_dtype=torch.float8_e4m3fn, **kw)
    new2, _ = gated_residual_norm(x, y, **kw)
    assert torch.equal(new, new2) and codes.shape == (M, K) and codes.dtype == torch.float8_e4m3fn
    _, hw, _, e2 = _want(x, y, gate, w2, b2, w1, b1, "rms", 0.5)
    pad = torch.nn.functional.pad(hw, (0, -K % 128)).view(M, -1, 128)
    amax = pad.abs().amax(2)
    assert ((scale.double() * 448 - amax).abs() <= e2 + amax * 2.0 ** -23).all()
    # half a step of E4M3: 2^-4 of the value, or half of the smallest step (2^-10) of the block's scale
    step = torch.maximum(hw.abs() * 2.0 ** -4, (amax / 448 * 2.0 ** -10).repeat_interleave(128, 1)[:, :K])
    d = dequantize_fp8_block(codes, scale).double()
    assert ((d - hw).abs() <= step * (1 + 2.0 ** -20) + 2 * e2).all()


def test_rows_without_variance_strided_and_empty():
    from vitfp4.nvfp4 import gated_residual_norm
    x = torch.full((3, 64), 2.0, device="cuda")
    new, h = gated_residual_norm(x, torch.ones_like(x))
    assert torch.equal(new, x) and torch.equal(h, torch.zeros_like(x))      # constant rows: 0 / sqrt(eps)
    new, h = gated_residual_norm(x[:, :1], x[:, 1:2])
    assert (new == 2).all() and (h == 0).all()
    big = torch.randn(40, 600, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    for a, b in ((big[:, 8:264], big[:, 300:556]), (big[:, 1:258], big[:, 3:260]), (big[::2, :100], big[1::2, 100:200])):
        got, want = gated_residual_norm(a, b), gated_residual_norm(a.contiguous(), b.contiguous())
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    e = big[:0]
    new, (c, s) = gated_residual_norm(e, e, out_dtype=torch.float8_e4m3fn)
    assert new.shape == (0, 600) and c.shape == (0, 600) and s.shape == (0, 5)
    n3, h3 = gated_residual_norm(big.view(4, 10, 600), big.flip(0).view(4, 10, 600))
    n2, h2 = gated_residual_norm(big, big.flip(0))
    assert torch.equal(n3.view(40, 600), n2) and torch.equal(h3.view(40, 600), h2)


def test_nan_stays_in_its_row_and_in_place_through_the_c_call():
    from vitfp4 import _lib
    from vitfp4.nvfp4 import gated_residual_norm
    g = torch.Generator(device="cuda").manual_seed(2)
    x, y = (torch.randn(50, 1016, device="cuda", generator=g).bfloat16() for _ in range(2))
    new, h = gated_residual_norm(x, y)
    bad = y.clone()
    bad[7, 3] = float("nan")
    n2, h2 = gated_residual_norm(x, bad)
    keep = torch.arange(50, device="cuda") != 7
    assert h2[7].isnan().all() and torch.equal(n2[keep], new[keep]) and torch.equal(h2[keep], h[keep])
    xi, hh = x.clone(), torch.empty_like(x)      # x_out is x
    _lib.call("vf4_gated_residual_norm", xi.data_ptr(), 1016, y.data_ptr(), 1016, 0, 50, 1016, None, 1, 1.0, 1, None, None, 1,
              None, None, 0, 1e-6, xi.data_ptr(), hh.data_ptr(), 0, 0, None, 0, 0, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(xi, new) and torch.equal(hh, h)


def test_too_long_rows_are_refused():
    from vitfp4 import _lib
    from vitfp4.nvfp4 import gated_residual_norm
    x = torch.zeros(2, 16385, device="cuda")
    with pytest.raises(_lib.VitFp4Error, match="16384"):
        gated_residual_norm(x, x)
