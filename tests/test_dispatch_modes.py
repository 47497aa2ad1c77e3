"""The FP8 block ops, the gated norm and cross attention under torch's dispatch modes: they go through their torch.library
ops there, as under torch.compile, so that fake tensors and tracers see them."""
import pytest
import torch

from vitfp4.nvfp4 import cross_sdpa, fp8_block_gemm, fp8_block_linear, gated_residual_norm, quantize_to_fp8_block

F8 = torch.float8_e4m3fn


def _calls(device):
    r = lambda *s: torch.randn(*s, device=device).bfloat16()
    x, w = r(2, 3, 200), torch.randn(140, 200, device=device).to(F8)
    ws = torch.rand(2, 2, device=device)
    buf = torch.randn(6, 208, device=device).to(F8)
    q, k = r(2, 3, 4, 64).transpose(1, 2), r(2, 2, 9, 64)
    mask = torch.rand(2, 9, device=device) < 0.5
    return {
        "vitfp4::cast_fp8_block": (lambda: quantize_to_fp8_block(x), [(2, 3, 200), (2, 3, 2)]),
        "vitfp4::linear_fp8_block": (lambda: fp8_block_linear(x, w, ws), [(2, 3, 140)]),
        "vitfp4::gemm_fp8_block": (lambda: fp8_block_gemm(buf[:, :200], torch.rand(6, 2, device=device), w, ws), [(6, 140)]),
        "vitfp4::gated_residual_norm": (lambda: gated_residual_norm(x, x, out_dtype=F8), [(2, 3, 200), (2, 3, 200), (2, 3, 2)]),
        "vitfp4::cross_attention": (lambda: cross_sdpa(q, k, k, key_mask=mask), [(2, 4, 3, 64)]),
    }


def _leaves(v):
    return [t for u in v for t in _leaves(u)] if isinstance(v, (tuple, list)) else [v]


NAMES = ["vitfp4::cast_fp8_block", "vitfp4::linear_fp8_block", "vitfp4::gemm_fp8_block", "vitfp4::gated_residual_norm",
         "vitfp4::cross_attention"]


@pytest.mark.parametrize("name", NAMES)
def test_fake_tensors(name):
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    with FakeTensorMode():
        call, shapes = _calls("cuda")[name]
        out = _leaves(call())
    assert [tuple(t.shape) for t in out] == shapes and all(isinstance(t, FakeTensor) for t in out)


def _seen(call):
    from torch.utils._python_dispatch import TorchDispatchMode
    names = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(func.name())
            return func(*args, **(kwargs or {}))

    with Watch():
        out = call()
    return names, out


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_mode_sees_the_op(name):
    torch.manual_seed(0)
    call, _ = _calls("cuda")[name]
    names, out = _seen(call)
    assert any(n.startswith(name) for n in names), names
    if name != "vitfp4::gemm_fp8_block":      # (its call draws scales)
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(_leaves(out), _leaves(call())))


@pytest.mark.gpu
def test_traced_calls_follow_their_inputs():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, y = torch.randn(2, 5, 256, device="cuda").bfloat16().unbind(0)
    f = lambda t: gated_residual_norm(t, t)[1]
    g = make_fx(f)(x)
    assert torch.equal(g(y), f(y)) and not torch.equal(g(y), f(x))
