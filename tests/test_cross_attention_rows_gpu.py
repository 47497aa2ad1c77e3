"""cross_sdpa where queries hold NaN or infinities and masks leave little or nothing, on each kernel."""
import math

import pytest
import torch
from test_cross_attention_gpu import _check, _inputs

pytestmark = pytest.mark.gpu

# a few rows over short keys (in one chunk, in several), many rows (in one, in several; 64 and 128 columns)
SHAPES = [(4, 2, 2, 1, 257, 64), (4, 1, 1, 1, 4000, 64), (4, 1, 1, 2, 500, 128), (4, 2, 2, 40, 300, 64), (4, 2, 1, 150, 515, 80), (4, 1, 1, 9, 5000, 128),
          (4, 1, 1, 33, 20000, 64), (4, 4, 2, 1, 5000, 128)]


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", SHAPES)
def test_a_query_that_keeps_no_key_gives_0_whatever_it_holds(B, H, Hkv, Sq, Skv, D, bad):
    from vitfp4 import _lib
    from vitfp4.nvfp4 import cross_sdpa
    q, k, v = _inputs(B, H, Hkv, Sq, Skv, D, seed=Skv, packed=True)
    keep = torch.rand(B, Skv, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) < 0.5
    keep[0] = False                        # nothing, by the mask
    keep[1, 130:] = False                  # nothing in later tiles and chunks
    keep[2, : Skv - 30] = False            # nothing in earlier ones
    want = cross_sdpa(q, k, v, key_mask=keep)
    _check(want, q, k, v, keep=keep)
    junk = q.clone()
    junk[0] = bad
    for b in (1, 2):
        junk[b, 0, Sq // 2, D - 3] = bad   # one query of images that keep some keys
    o = cross_sdpa(junk, k, v, key_mask=keep)
    assert (o[0] == 0).all()
    assert o[1, 0, Sq // 2].isnan().all() and o[2, 0, Sq // 2].isnan().all()
    for b in (1, 2):
        o[b, 0, Sq // 2] = want[b, 0, Sq // 2]
    assert torch.equal(o, want)
    lens = torch.tensor([0, Skv, 0, 130], dtype=torch.int32, device="cuda")
    full = torch.ones_like(keep)
    o = cross_sdpa(torch.full_like(q, bad), k, v, kv_lens=lens, key_mask=full)
    assert (o[0] == 0).all() and (o[2] == 0).all() and o[1].isnan().all() and o[3].isnan().all()
    full[1] = False
    o = cross_sdpa(torch.full_like(q, bad), k, v, kv_lens=lens, key_mask=full)
    assert (o[:3] == 0).all() and o[3].isnan().all()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", SHAPES)
def test_kept_scores_of_minus_infinity_are_no_dropped_keys(B, H, Hkv, Sq, Skv, D, masked):
    """Scores below the lowest finite number: a row of them is NaN, as softmax gives it; beside finite ones they weigh 0.
    Keys and queries are powers of two, so that every sum is exact or overflows whatever its order."""
    from vitfp4.nvfp4 import cross_sdpa
    _, _, v = _inputs(B, H, Hkv, Sq, Skv, D, seed=Skv)
    q = torch.full((B, H, Sq, D), 2.0 ** 70, device="cuda").bfloat16()
    k = torch.full((B, Hkv, Skv, D), -(2.0 ** 70), device="cuda").bfloat16()      # scores -2^140 D: -inf
    keep = torch.ones(B, Skv, dtype=torch.bool, device="cuda")
    if masked:
        keep[:, 5::3] = False
    kw = dict(key_mask=keep) if masked else {}
    assert cross_sdpa(q, k, v, **kw).isnan().all()
    k2 = k.clone()
    for at in (0, Skv - 1):          # one key with a score of 0: its value alone
        k2[:] = k
        k2[:, :, at] = 0
        keep[:, at] = True
        o = cross_sdpa(q, k2, v, **kw)
        assert torch.equal(o, v[:, :, at, None].repeat_interleave(H // Hkv, 1).expand(B, H, Sq, D))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", SHAPES)
def test_kept_scores_near_the_lowest_number(B, H, Hkv, Sq, Skv, D, masked):
    """All scores between -2^127 and -2^126 (times a scale that brings them to -2 .. -1): weights as any others."""
    from vitfp4.nvfp4 import cross_sdpa
    _, _, v = _inputs(B, H, Hkv, Sq, Skv, D, seed=Skv)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.zeros(B, H, Sq, D, device="cuda").bfloat16()
    k = torch.zeros(B, Hkv, Skv, D, device="cuda").bfloat16()
    q[..., 1] = 2.0 ** 63            # one product per score: no sum to round
    k[..., 1] = (-(2.0 ** 63) * (1 + torch.rand(B, Hkv, Skv, device="cuda", generator=g) * 0.98)).bfloat16()
    keep = torch.ones(B, Skv, dtype=torch.bool, device="cuda")
    if masked:
        keep[:, 5::3] = False
    o = cross_sdpa(q, k, v, scale=2.0 ** -126, **(dict(key_mask=keep) if masked else {}))
    _check(o, q, k, v, scale=2.0 ** -126, keep=keep)


@pytest.mark.parametrize("Sq,Skv,D", [(1, 40, 64), (1, 1, 64), (30, 200, 64), (1, 6000, 128), (140, 1, 80)])
def test_strides_of_single_entries_mean_nothing(Sq, Skv, D):
    """One image, one head, one query or one key with a stride that is no multiple of 8 elements."""
    from vitfp4.nvfp4 import cross_sdpa, ops
    for H, Hkv in ((2, 2), (2, 1), (1, 1)):
        q, k, v = _inputs(1, H, Hkv, Sq, Skv, D, seed=Sq)
        want = cross_sdpa(q, k, v)

        def odd(t):
            strides = [s + 1 if n == 1 else s for n, s in zip(t.shape, t.contiguous().stride())]
            return t.new_zeros(t.numel() + 8).as_strided(t.shape, strides).copy_(t)

        qo, ko, vo = odd(q), odd(k), odd(v)
        assert qo.stride(0) % 8 and ko.stride(0) % 8
        assert torch.equal(cross_sdpa(qo, ko, vo), want)
        ops.probe.timing = True          # the Python path
        try:
            assert torch.equal(cross_sdpa(qo, ko, vo), want)
        finally:
            ops.probe.timing = False
            ops.probe.reset()


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("power", [4, 10, 17, 22, 40])
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", SHAPES)
def test_huge_scores_pick_the_key_of_the_largest(B, H, Hkv, Sq, Skv, D, power, sign):
    """Scores of 2^(2 power) times whole numbers below 256, exact in fp32 whatever the order: the largest stands at least
    2^(2 power) above the next one, so its value comes out alone, rounded by nothing."""
    from vitfp4.nvfp4 import cross_sdpa
    _, _, v = _inputs(B, H, Hkv, Sq, Skv, D, seed=Skv)
    g = torch.Generator(device="cuda").manual_seed(power)
    n = torch.randint(20, 180, (B, Hkv, Skv), device="cuda", generator=g).float()
    q = torch.zeros(B, H, Sq, D, device="cuda").bfloat16()
    k = torch.zeros(B, Hkv, Skv, D, device="cuda").bfloat16()
    q[..., 3] = sign * 2.0 ** power
    keep = torch.ones(B, Skv, dtype=torch.bool, device="cuda")
    keep[:, 7::5] = False
    for at in (0, Skv // 2 // 5 * 5, Skv - 1):
        m = n.clone()
        m[:, :, at] = 190.0 if sign > 0 else 10.0
        k[..., 3] = (m * 2.0 ** power).bfloat16()
        keep[:, at] = True
        want = v[:, :, at, None].repeat_interleave(H // Hkv, 1).expand(B, H, Sq, D)
        for kw in ({}, {"key_mask": keep}):
            o = cross_sdpa(q, k, v, scale=1.0, **kw)
            # (the largest weight may be the polynomial's 2^0, off by 2^-20: half a step of bf16 covers it)
            assert torch.equal(o, want), (at, float((o.float() - want.float()).abs().max()))
