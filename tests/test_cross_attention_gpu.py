"""cross_sdpa on the GPU against exact attention in 64 bits.

Tolerance, for scores bounded by S (largest |scale q.k| in units of log2) and values bounded by V.  A score is a sum of
D exact products in fp32, off by at most D 2^-23 of the sum of magnitudes (in log2 units e_s = D 2^-23 * scale * log2 e *
sum |q||k|, plus two roundings of S * 2^-24 in the exponent's fused multiply-add); 2^x multiplies that by ln 2 and adds
the special-function unit's 2^-22: a weight is off by a relative e_w = 0.7 (e_s + 4 S 2^-24) + 2^-22.  The tensor-core
kernel rounds weights to bf16 for the product with the values (half a step, 2^-9 relative to the weight's leading power
of two, at most 2^-8 of the weight) but sums them unrounded; the sums over keys are off by Skv 2^-23 at most.  So
|err| <= (2 e_w + 2^-8 + 4 Skv 2^-23) sum_j p_j |v_j| / sum_j p_j, and half a bf16 step (2^-8 relative) of the result.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(B, H, Hkv, Sq, Skv, D, seed=0, packed=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    q = r(B, Sq, H, D).transpose(1, 2)
    if packed:   # K and V as views of one projection
        kv = r(B, Skv, 2, Hkv, D)
        return q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    return q, r(B, Hkv, Skv, D), r(B, Hkv, Skv, D)


def _exact(q, k, v, scale, keep):
    """(output, weighted sum of |v|, largest |score|, largest sum of |q||k|) in 64 bits; keep (B, Skv) bool."""
    B, H, Sq, D = q.shape
    G = H // k.shape[1]
    kk, vv = (t.double().repeat_interleave(G, 1) for t in (k, v))
    kk, vv = (torch.where(keep[:, None, :, None], t, 0.0) for t in (kk, vv))
    s = q.double() @ kk.transpose(2, 3) * scale
    mag = (q.double().abs() @ kk.abs().transpose(2, 3)).amax() * abs(scale) if kk.shape[2] and Sq else torch.zeros(())
    s = s.masked_fill(~keep[:, None, None, :], -math.inf)
    top = s.amax(3, keepdim=True) if s.shape[3] else torch.zeros(B, H, Sq, 1, device=q.device, dtype=torch.float64)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    t = p.sum(3, keepdim=True)
    t = torch.where(t > 0, t, 1.0)
    return p @ vv / t, p @ vv.abs() / t, float(mag)


def _check(o, q, k, v, scale=None, keep=None):
    B, H, Sq, D = q.shape
    Skv = k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    keep = torch.ones(B, Skv, dtype=torch.bool, device="cuda") if keep is None else keep
    want, mag, s = _exact(q, k, v, scale, keep)
    s2 = s * 1.4427
    e_w = 0.7 * (D * 2.0 ** -23 * s2 + 4 * s2 * 2.0 ** -24) + 2.0 ** -22
    tol = (2 * e_w + 2.0 ** -8 + 4 * max(Skv, 1) * 2.0 ** -23) * mag + want.abs() * 2.0 ** -8 * 1.001 + 1e-30
    assert o.shape == q.shape and o.dtype == torch.bfloat16
    bad = ~((o.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((o.double() - want).abs() / tol).max()))


SHAPES = [  # B, H, Hkv, Sq, Skv, D
    (1, 1, 1, 1, 1, 64), (2, 3, 3, 1, 257, 64), (2, 4, 2, 1, 130, 32), (1, 8, 2, 1, 1000, 128), (3, 2, 2, 3, 77, 80), (1, 2, 1, 2, 5000, 96),
    (2, 2, 2, 5, 1, 64), (1, 3, 3, 17, 127, 64), (2, 2, 2, 64, 1025, 80), (1, 8, 2, 4, 300, 128), (2, 1, 1, 128, 128, 64), (1, 2, 2, 129, 129, 72),
    (1, 2, 2, 200, 400, 128), (1, 1, 1, 256, 640, 8), (2, 2, 1, 300, 260, 40), (1, 1, 1, 1000, 33, 104), (1, 4, 1, 70, 515, 64), (1, 1, 1, 33, 20000, 64),
    (1, 1, 1, 300, 9000, 128), (40, 4, 4, 20, 150, 64), (1, 12, 12, 385, 385, 64)]


@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", SHAPES)
def test_matches_exact_attention(B, H, Hkv, Sq, Skv, D):
    from vitfp4 import _lib
    from vitfp4.nvfp4 import cross_sdpa
    q, k, v = _inputs(B, H, Hkv, Sq, Skv, D, seed=Sq + Skv)
    o = cross_sdpa(q, k, v)
    _check(o, q, k, v)
    assert torch.equal(o, cross_sdpa(q, k, v))
    assert _lib.device_error() == 0


@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", [(6, 2, 2, 1, 700, 64), (6, 4, 1, 1, 3000, 128), (6, 2, 2, 40, 300, 64), (6, 2, 1, 150, 515, 80),
                                             (6, 1, 1, 9, 5000, 128), (6, 1, 1, 260, 129, 128)])
@pytest.mark.parametrize("kind", ["lens", "mask", "both"])
def test_masked_keys_may_hold_anything(B, H, Hkv, Sq, Skv, D, kind):
    from vitfp4.nvfp4 import cross_sdpa
    q, k, v = _inputs(B, H, Hkv, Sq, Skv, D, seed=Skv, packed=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = torch.tensor([Skv, 0, 1, Skv // 2, 128, Skv + 5], dtype=torch.int32, device="cuda") if kind != "mask" else None
    keep = torch.ones(B, Skv, dtype=torch.bool, device="cuda")
    mask = None
    if kind != "lens":
        mask = torch.rand(B, Skv, device="cuda", generator=g) < 0.6
        mask[2] = False                     # an image whose mask leaves nothing
        mask[4, : min(Skv, 256)] = False    # whole tiles without a key
        mask[5] = True
        keep &= mask
    if lens is not None:
        keep &= torch.arange(Skv, device="cuda")[None] < lens[:, None]
    drop = ~keep[:, None, :, None]
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda").bfloat16()
    junk = bad[torch.arange(k.numel(), device="cuda").view(k.shape) % 4]
    kj, vj = torch.where(drop, junk, k), torch.where(drop, junk, v)
    o = cross_sdpa(q, kj, vj, kv_lens=lens, key_mask=mask)
    _check(o, q, k, v, keep=keep)
    empty = ~keep.any(1)
    assert empty.any() and (o[empty] == 0).all()
    clean = cross_sdpa(q, torch.where(drop, 0, k), torch.where(drop, 0, v), kv_lens=lens, key_mask=mask)
    assert torch.equal(o, clean)
    if lens is not None and mask is None:
        assert torch.equal(o, cross_sdpa(q, kj, vj, kv_lens=lens.long()))


@pytest.mark.parametrize("scale", [0.5, -0.3, 0.0, 3.0])
@pytest.mark.parametrize("Sq", [1, 30, 200])
def test_scales_of_any_sign(scale, Sq):
    from vitfp4.nvfp4 import cross_sdpa
    q, k, v = _inputs(2, 2, 1, Sq, 333, 64, seed=5)
    lens = torch.tensor([333, 100], device="cuda", dtype=torch.int32)
    keep = torch.arange(333, device="cuda")[None] < lens[:, None]
    _check(cross_sdpa(q, k, v, scale=scale, kv_lens=lens), q, k, v, scale=scale, keep=keep)


@pytest.mark.parametrize("Sq", [2, 20, 140])
def test_scores_that_grow_along_the_keys(Sq):
    """Maxima that move by more and by less than the kernel's threshold from tile to tile, both ways."""
    from vitfp4.nvfp4 import cross_sdpa
    for seed, ramp in ((0, torch.linspace(-4, 4, 1300)), (1, torch.linspace(4, -4, 1300)), (2, torch.linspace(-0.2, 0.2, 1300)),
                       (3, 3 * torch.sin(torch.arange(1300) / 90.0))):
        q, k, v = _inputs(1, 2, 2, Sq, 1300, 64, seed=seed)
        q = (q.abs() + 0.5).bfloat16()
        k = (k * 0.1 + ramp.cuda()[None, None, :, None]).bfloat16()
        _check(cross_sdpa(q, k, v), q, k, v)


def test_strides_broadcasts_and_nan_rows():
    from vitfp4.nvfp4 import cross_sdpa
    for Sq in (1, 50, 130):
        q, k, v = _inputs(3, 4, 2, Sq, 200, 64, seed=7)
        want = cross_sdpa(q, k, v)
        lat = q[:1].expand(3, -1, -1, -1)                     # one set of latents for the batch
        o = cross_sdpa(lat, k, v)
        _check(o, lat, k, v)
        one = cross_sdpa(q, k[:1].expand(3, -1, -1, -1), v[:, :1].expand(-1, 2, -1, -1))
        _check(one, q, k[:1].expand(3, -1, -1, -1), v[:, :1].expand(-1, 2, -1, -1))
        odd = torch.zeros(3, 2, 200, 67, device="cuda", dtype=torch.bfloat16)
        odd[..., 1:65] = k                                     # misaligned rows are copied
        assert torch.equal(cross_sdpa(q, odd[..., 1:65], v), want)
        assert torch.equal(cross_sdpa(q.transpose(2, 3).contiguous().transpose(2, 3), k, v), want)
        assert want.transpose(1, 2).is_contiguous()
        bad = q.clone()
        bad[1, 2, Sq // 2, 5] = float("nan")
        o = cross_sdpa(bad, k, v)
        assert o[1, 2, Sq // 2].isnan().all()
        o[1, 2, Sq // 2] = want[1, 2, Sq // 2]
        assert torch.equal(o, want)
        v2 = v.clone()
        v2[0, 0, 17, 3] = float("inf")
        o = cross_sdpa(q, k, v2)
        assert o[0, :2, :, 3].isinf().all() and torch.equal(o[1:], want[1:]) and torch.equal(o[0, 2:], want[0, 2:])


def test_no_keys_no_queries_no_images():
    from vitfp4.nvfp4 import cross_sdpa
    for Sq in (1, 3, 300):
        q, k, v = _inputs(2, 4, 2, Sq, 9, 64)
        assert (cross_sdpa(q, k[:, :, :0], v[:, :, :0]) == 0).all()
        assert cross_sdpa(q[:, :, :0], k, v).shape == (2, 4, 0, 64)
        assert cross_sdpa(q[:0], k[:0], v[:0]).shape == (0, 4, Sq, 64)


def test_captured_replayed_and_on_two_streams():
    from vitfp4.nvfp4 import cross_sdpa
    for Sq, Skv in ((1, 6000), (40, 6000), (150, 300)):      # the first two with partial results in a workspace
        sets = [_inputs(1, 2, 2, Sq, Skv, 64, seed=i) for i in range(3)]
        want = [cross_sdpa(*s) for s in sets]
        streams = [torch.cuda.Stream() for _ in range(3)]
        got = []
        for st, s in zip(streams, sets):                     # calls that overlap share nothing
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(cross_sdpa(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        buf = [t.clone() for t in sets[0]]
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        outs = []
        for gr in graphs:
            with torch.cuda.graph(gr):
                outs.append(cross_sdpa(*buf))
        for s, w in zip(sets, want):
            for b, t in zip(buf, s):
                b.copy_(t)
            for gr in graphs:
                gr.replay()
            assert torch.equal(outs[0], w) and torch.equal(outs[1], w)


def test_workspace_is_checked():
    from vitfp4 import _lib
    q, k, v = _inputs(1, 2, 2, 1, 6000, 64)
    o = torch.full((1, 1, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    n = _lib.lib().vf4_cross_attn_workspace_size(1, 2, 2, 1, 6000, 64)
    assert n > 0
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    args = lambda bytes_: (q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], 1, 2, 2, 1, 6000,
                           64, 0.125, None, None, 0, o.data_ptr(), 128, 64, 128, ws.data_ptr(), bytes_, torch.cuda.current_stream().cuda_stream)
    with pytest.raises(_lib.VitFp4Error, match="workspace"):
        _lib.call("vf4_cross_attn", *args(n - 1))
    torch.cuda.synchronize()
    assert (o == 7).all()
    _lib.call("vf4_cross_attn", *args(n))
    assert (o != 7).any()
