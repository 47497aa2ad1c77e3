"""The C++ form of the small ops' plain calls (vitfp4._fast): what it leaves to the Python path (no GPU), and that both
paths launch the same kernels (GPU)."""
import pytest
import torch

from vitfp4.nvfp4 import ops

F8 = torch.float8_e4m3fn


def _module():
    if ops._fast_module is None:
        pytest.skip("vitfp4/_fast.so is not built (run __graft_entry__.build())")
    return ops._fast_module


def test_everything_but_plain_cuda_tensors_is_left_alone():
    m = _module()
    x, w, s = torch.zeros(2, 32), torch.zeros(4, 32).to(F8), torch.ones(1, 1)
    for fn, args in ((m.cast, (x,)), (m.linear, (x, w, s, None)), (m.norm, (x, x, None, 1.0, 1, None, None, None, None, 1e-6, False)),
                     (m.cross, (x, x, x, None, None, None))):
        assert fn(*args) is None                       # CPU tensors
        assert fn(*args[:-1]) is None and fn() is None  # another number of arguments
        assert fn(*[None] * len(args)) is None
        assert fn(*["x"] * len(args)) is None


def _calls():
    from vitfp4 import nvfp4 as api
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, y = r(6, 256).bfloat16(), r(6, 256).bfloat16()
    many = r(90, 256).bfloat16()
    w, ws = api.quantize_to_fp8_block(r(64, 256), 128)
    bias, gate, nw = r(64).bfloat16(), r(3, 256).bfloat16(), r(256).bfloat16()
    q, kv = r(2, 5, 4, 64).bfloat16().transpose(1, 2), r(2, 400, 2, 2, 64).bfloat16()
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    lens, mask = torch.tensor([400, 3], dtype=torch.int32, device="cuda"), r(2, 400) > 0
    return [
        ("cast", 1, lambda: api.quantize_to_fp8_block(x)),
        ("cast f32", 1, lambda: api.quantize_to_fp8_block(x.float())),
        ("linear one", 1, lambda: api.fp8_block_linear(x[:1], w, ws, bias=bias)),
        ("linear few", 2, lambda: api.fp8_block_linear(x[:3], w, ws, bias=bias)),
        ("linear", 2, lambda: api.fp8_block_linear(many, w, ws)),
        ("linear f32", 2, lambda: api.fp8_block_linear(many.float(), w, ws, bias=bias.float())),
        ("norm", 1, lambda: api.gated_residual_norm(x, y, gate=gate, residual_scale=0.5, post_weight=nw, pre_weight=nw, pre_bias=nw)),
        ("norm rms f32", 1, lambda: api.gated_residual_norm(x.float(), y.float(), norm="rms")),
        ("norm fp8", 1, lambda: api.gated_residual_norm(x, y, gate=gate[0], pre_weight=nw, out_dtype=F8)),
        ("cast 3d", 1, lambda: api.quantize_to_fp8_block(x.view(2, 3, 256))),
        ("linear 4d", 2, lambda: api.fp8_block_linear(many.view(3, 5, 6, 256), w, ws, bias=bias)),
        ("norm 3d", 1, lambda: api.gated_residual_norm(x.view(3, 2, 256), y.view(3, 2, 256), gate=gate, norm="rms")),
        ("norm fp8 3d", 1, lambda: api.gated_residual_norm(x.view(3, 2, 256), y.view(3, 2, 256), out_dtype=F8)),
        ("cast odd", 1, lambda: api.quantize_to_fp8_block(x.float()[:, :201])),
        ("cast odd 3d", 1, lambda: api.quantize_to_fp8_block(x[:, :130].reshape(2, 3, 130).contiguous())),
        ("linear odd", 2, lambda: api.fp8_block_linear(many[:, :201], *api.quantize_to_fp8_block(many[:64, :201], 128))),
        ("norm fp8 odd 3d", 1, lambda: api.gated_residual_norm(*[t[:, :201].reshape(2, 3, 201).contiguous() for t in (x, y)], out_dtype=F8)),
        ("cross", 1, lambda: api.cross_sdpa(q, k, v, kv_lens=lens, scale=0.2)),
        ("cross mask", 1, lambda: api.cross_sdpa(q, k, v, key_mask=mask)),
        ("cross chunks", 2, lambda: api.cross_sdpa(q, k.repeat(1, 1, 3, 1), v.repeat(1, 1, 3, 1))),
    ]


def _leaves(v):
    return [t for u in v for t in _leaves(u)] if isinstance(v, (tuple, list)) else [v]


@pytest.mark.gpu
def test_both_paths_give_the_same(monkeypatch):
    m = _module()
    taken = []
    for name, launches, call in _calls():
        ops.probe.reset()
        plain = _leaves(call())
        n = ops.probe.launches
        assert m.launched() == launches and n >= launches, name
        ops.probe.timing = True     # the probe's calls go the Python way
        try:
            python = _leaves(call())
        finally:
            ops.probe.timing = False
        assert len(plain) == len(python), name
        for a, b in zip(plain, python):
            assert a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride(), name
            assert torch.equal(a.float(), b.float()), name
        taken.append(name)
    assert len(ops.probe.records) and len(taken) == 20
    ops.probe.reset()


@pytest.mark.gpu
def test_calls_that_are_not_plain_go_the_python_way():
    from vitfp4 import nvfp4 as api
    m = _module()
    x = torch.randn(6, 100, device="cuda").bfloat16()
    assert m.cast(x) is not None and m.cast(x[:, ::2]) is None  # columns apart
    assert m.cast(x.t()) is None and m.cast(x[:0]) is None     # copies, nothing to do
    p = torch.nn.Parameter(torch.randn(4, 128, device="cuda"))
    assert m.cast(p) is None                                   # gradients recorded
    with torch.no_grad():
        assert m.cast(p) is not None
    q = torch.randn(2, 4, 3, 64, device="cuda").bfloat16()
    assert m.cross(q, q[:, :3], q[:, :3], None, None, None) is None        # 4 heads over 3
    assert m.cross(q, q, q, None, None, float("nan")) is None
    assert m.cross(q[..., 1:33], q[..., 1:33], q[..., 1:33], None, None, None) is None
    y = torch.randn(6, 128, device="cuda")
    for kind in (0, 3):
        assert m.norm(y, y, None, 1.0, kind, None, None, None, None, 1e-6, False) is None
    with pytest.raises(Exception):
        api.gated_residual_norm(y, y, norm=None)


@pytest.mark.gpu
def test_calls_that_only_look_alike():
    from vitfp4 import _lib
    from vitfp4 import nvfp4 as api
    x = torch.randn(2, 3, 256, device="cuda").bfloat16()
    w, ws = api.quantize_to_fp8_block(torch.randn(64, 256, device="cuda"), 128)
    with pytest.raises(_lib.VitFp4Error):      # as many rows, another shape
        api.gated_residual_norm(x, x.view(3, 2, 256))
    turned = x.transpose(0, 1)                 # not contiguous: rows in another order
    assert torch.equal(api.fp8_block_linear(turned, w, ws), api.fp8_block_linear(turned.contiguous(), w, ws))
    assert torch.equal(api.gated_residual_norm(turned, turned)[1], api.gated_residual_norm(turned.contiguous(), turned.contiguous())[1])
    empty = x[:, :0]
    assert api.fp8_block_linear(empty, w, ws).shape == (2, 0, 64) and api.quantize_to_fp8_block(empty)[1].shape == (2, 0, 2)
    assert api.gated_residual_norm(empty, empty, out_dtype=F8)[1][1].shape == (2, 0, 2)
    one = x[0, 0]
    assert torch.equal(api.fp8_block_linear(one, w, ws), api.fp8_block_linear(one[None], w, ws)[0])
