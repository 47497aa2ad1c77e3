"""FP8 block format: refusals and the format's helpers (no GPU)."""
import pytest
import torch

from vitfp4 import _lib
from vitfp4.nvfp4 import dequantize_fp8_block, fp8_block_gemm, fp8_block_linear, quantize_to_fp8_block

F8 = torch.float8_e4m3fn


def _op(rows, K, block_rows):
    return torch.zeros(rows, K).to(F8), torch.ones(-(-rows // block_rows), -(-K // 128))


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.VitFp4Error, match="CUDA"):
        quantize_to_fp8_block(torch.zeros(2, 128))
    with pytest.raises(_lib.VitFp4Error, match="CUDA"):
        fp8_block_gemm(*_op(3, 128, 1), *_op(5, 128, 128))
    with pytest.raises(_lib.VitFp4Error, match="CUDA"):
        fp8_block_linear(torch.zeros(3, 128), *_op(5, 128, 128))


def test_block_rows_and_rank_are_checked():
    with pytest.raises(_lib.VitFp4Error, match="block_rows"):
        quantize_to_fp8_block(torch.zeros(2, 128), 64)
    with pytest.raises(_lib.VitFp4Error, match="2-D weight"):
        quantize_to_fp8_block(torch.zeros(2, 2, 128), 128)


@pytest.mark.parametrize("bad", ["codes dtype", "scale shape", "scale dtype", "k", "bias shape", "bias strides", "out dtype", "empty weight"])
def test_product_arguments_are_checked(bad):
    a, sa = _op(3, 256, 1)
    b, sb = _op(130, 256, 128)
    bias, kw = None, {}
    if bad == "codes dtype":
        a = a.view(torch.uint8)
    elif bad == "scale shape":
        sb = sb[:1]
    elif bad == "scale dtype":
        sa = sa.double()
    elif bad == "k":
        b, sb = _op(130, 128, 128)
    elif bad == "bias shape":
        bias = torch.zeros(129)
    elif bad == "bias strides":
        bias = torch.zeros(260)[::2]
    elif bad == "out dtype":
        kw["out_dtype"] = torch.float16
    else:
        b, sb = _op(0, 256, 128)
    with pytest.raises(_lib.VitFp4Error):
        fp8_block_gemm(a, sa, b, sb, bias=bias, **kw)
    if bad in ("scale shape", "k", "bias shape", "bias strides", "empty weight"):
        with pytest.raises(_lib.VitFp4Error):
            fp8_block_linear(torch.zeros(3, 256), b, sb, bias=bias)


def test_dequantize_activation_and_weight_blocks():
    codes = torch.full((130, 200), 2.0).to(F8)
    act = torch.arange(260.0).view(130, 2)
    d = dequantize_fp8_block(codes, act)
    assert torch.equal(d[:, :128], 2 * act[:, :1].expand(130, 128)) and torch.equal(d[:, 128:], 2 * act[:, 1:].expand(130, 72))
    w = torch.tensor([[1.0, 2.0], [3.0, 4.0]])
    d = dequantize_fp8_block(codes, w)
    assert d[0, 0] == 2 and d[127, 199] == 4 and d[128, 0] == 6 and d[129, 128] == 8


def test_codes_of_more_dimensions_are_checked():
    a, sa = _op(6, 256, 1)
    b, sb = _op(130, 256, 128)
    with pytest.raises(_lib.VitFp4Error, match="CUDA"):                    # taken, as far as there is a GPU
        fp8_block_gemm(a.view(2, 3, 256), sa.view(2, 3, 2), b, sb)
    for codes, scale in ((a.view(2, 3, 256), sa), (a.view(2, 3, 256), sa.view(3, 2, 2)), (a.view(2, 3, 256), torch.ones(2, 3, 1)),
                         (a.view(2, 3, 256), torch.tensor(1.0)), (a[0, 0], sa[0, 0]), (a[:, :0].view(2, 3, 0), sa[:, :0].view(2, 3, 0))):
        with pytest.raises(_lib.VitFp4Error) as e:
            fp8_block_gemm(codes, scale, b, sb)
        assert "CUDA" not in str(e.value)


def test_inputs_without_columns_are_refused():
    w, ws = _op(5, 128, 128)
    for x in (torch.tensor(1.0), torch.zeros(2, 3, 0), torch.zeros(0)):
        with pytest.raises(_lib.VitFp4Error):
            quantize_to_fp8_block(x)
        with pytest.raises(_lib.VitFp4Error):
            fp8_block_linear(x, w, ws)
