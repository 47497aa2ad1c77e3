"""The FP8 block ops, the gated residual norm and cross attention run together: a cross-attention block of latents over a
ViT's tokens, as a resampler or a pooling head uses them.

    x0, h  = norms of the latents (pre-norm, FP8)          kv = fp8_linear(tokens)
    q      = fp8_gemm(h)                                    o = cross_sdpa(q, k, v, token counts)
    a      = fp8_linear(o)
    x1, h1 = x0 + 0.5 gate N(a), N(x1) in FP8              f = fp8_gemm(h1), x2 = x1 + 0.5 gate N(f)

Against the same block in 64 bits without quantization: an E4M3 operand is off by at most half a step, 2^-4 of each value
(2^-4 / sqrt 3 in the mean square of a uniform error, 0.036); two operands per product make 0.05 of its output's norm where
signs are random, the longest path has four products (kv, attention output, h1, and q beside kv), 0.2 in all with each
norm passing relative errors on; the residual x0, which is exact, is more than half of the result: 0.2 bounds it.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
B, L, T, D, H, HKV, HD = 3, 20, 197, 256, 4, 2, 64


def _weights(seed=0):
    from vitfp4.nvfp4 import quantize_to_fp8_block
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    w = {"q": r(H * HD, D) / D ** 0.5, "kv": r(2 * HKV * HD, D) / D ** 0.5, "o": r(D, H * HD) / (H * HD) ** 0.5, "f": r(D, D) / D ** 0.5}
    p = {"full": {k: v.double() for k, v in w.items()}, "fp8": {k: quantize_to_fp8_block(v, 128) for k, v in w.items()}}
    p["bias"] = r(2 * HKV * HD).bfloat16()
    p["gate"] = r(B, D).bfloat16()
    p["w"] = (1 + 0.1 * r(D)).bfloat16()
    return p


def _inputs(seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, L, D, device="cuda", generator=g).bfloat16()
    t = torch.randn(B, T, D, device="cuda", generator=g).bfloat16()
    return x, t, torch.tensor([T, 50, 0], dtype=torch.int32, device="cuda")


def _block(p, x, tokens, lens):
    from vitfp4.nvfp4 import cross_sdpa, fp8_block_gemm, fp8_block_linear, gated_residual_norm
    x0, (hc, hs) = gated_residual_norm(x, None, norm="rms", pre_weight=p["w"], out_dtype=F8)
    q = fp8_block_gemm(hc.reshape(B * L, D), hs.reshape(B * L, -1), *p["fp8"]["q"]).view(B, L, H, HD).transpose(1, 2)
    kv = fp8_block_linear(tokens, *p["fp8"]["kv"], bias=p["bias"]).view(B, T, 2, HKV, HD)
    o = cross_sdpa(q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), kv_lens=lens)
    a = fp8_block_linear(o.transpose(1, 2).reshape(B, L, H * HD), *p["fp8"]["o"])
    kw = dict(gate=p["gate"], residual_scale=0.5, norm="rms", post_weight=p["w"])
    x1, (hc, hs) = gated_residual_norm(x0, a, pre_weight=p["w"], out_dtype=F8, **kw)
    f = fp8_block_gemm(hc.reshape(B * L, D), hs.reshape(B * L, -1), *p["fp8"]["f"]).view(B, L, D)
    x2, _ = gated_residual_norm(x1, f, pre_norm=False, **kw)
    return x2


def _exact(p, x, tokens, lens):
    w = {k: v for k, v in p["full"].items()}
    n = lambda v: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * p["w"].double()
    x, tokens, gate = x.double(), tokens.double(), p["gate"].double()[:, None]
    q = (n(x) @ w["q"].t()).view(B, L, H, HD).transpose(1, 2)
    kv = (tokens @ w["kv"].t() + p["bias"].double()).view(B, T, 2, HKV, HD)
    k, v = (kv[:, :, i].transpose(1, 2).repeat_interleave(H // HKV, 1) for i in (0, 1))
    s = (q @ k.transpose(2, 3) * HD ** -0.5).masked_fill(~(torch.arange(T, device="cuda") < lens[:, None])[:, None, None], -torch.inf)
    o = torch.nan_to_num(torch.softmax(s, 3)) @ v
    a = o.transpose(1, 2).reshape(B, L, H * HD) @ w["o"].t()
    x1 = x + 0.5 * gate * n(a)
    return x1 + 0.5 * gate * n(n(x1) @ w["f"].t())


def test_block_against_64_bits():
    p, (x, t, lens) = _weights(), _inputs()
    got, want = _block(p, x, t, lens).double(), _exact(p, x, t, lens)
    assert float((got - want).norm() / want.norm()) < 0.2
    assert torch.equal(got, _block(p, x, t, lens).double())


def test_block_captured_on_a_side_stream_and_replayed_on_new_inputs():
    from vitfp4 import _lib
    p, (x, t, lens) = _weights(), _inputs()
    _block(p, x, t, lens)
    bx, bt, bl = x.clone(), t.clone(), lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = _block(p, bx, bt, bl)
    for seed in (1, 5, 6):
        x, t, lens = _inputs(seed)
        bx.copy_(x), bt.copy_(t), bl.copy_(lens.flip(0))
        graph.replay()
        assert torch.equal(out, _block(p, x, t, lens.flip(0)))
    assert _lib.device_error() == 0


def test_block_traces_and_says_that_it_has_no_backward():
    p, (x, t, lens) = _weights(), _inputs()
    want = _block(p, x, t, lens)
    with torch.no_grad():
        got = torch.compile(lambda a, b, c: _block(p, a, b, c), backend="eager", fullgraph=True)(x, t, lens)
    assert torch.equal(got, want)
    xg = x.clone().requires_grad_()
    y = _block(p, xg, t, lens)
    assert torch.equal(y, want) and y.requires_grad
    with pytest.raises(Exception):
        y.float().sum().backward()
