"""FP8 block format: E4M3 codes with one fp32 scale per block of 128, and the product of two such operands.

The 8-bit step between the NVFP4 path and bf16, for layers a policy keeps out of NVFP4 (heads, first and last
blocks, the projections of a cross attention).  No counterpart in the reference, whose 8-bit format is a per-row
round trip inside attention (src/vit_nvfp4/nvfp4/fp8.py:6-17).

    amax' = max(amax |x| over the block, 1e-12)
    scale = amax' / 448,   code = e4m3(448 x / amax')          (decode: code * scale)

Activations have a block per 128 consecutive columns of a row, weights per 128 x 128 block.  Codes live in rows
padded to 16 bytes (the returned tensor is a view of the first K columns), so any K works.  Inference only: the
ops have no backward pass.
"""
from __future__ import annotations

import torch

from .. import _lib
from . import ops

_BLOCK = 128
_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _check_operand(name: str, codes: torch.Tensor, scale: torch.Tensor, block_rows: int) -> None:
    if codes.dtype != torch.float8_e4m3fn or codes.dim() != 2:
        raise _lib.VitFp4Error(f"{name}: (rows, K) float8_e4m3fn codes needed, got {tuple(codes.shape)} {codes.dtype}")
    rows, K = codes.shape
    want = ((rows + block_rows - 1) // block_rows, (K + _BLOCK - 1) // _BLOCK)
    if scale.dtype != torch.float32 or scale.shape != want:
        raise _lib.VitFp4Error(f"{name}: scales of {tuple(codes.shape)} codes are {want} fp32, got {tuple(scale.shape)} "
                               f"{scale.dtype}")


def _check_weight(w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None) -> None:
    _check_operand("weight", w, w_scale, _BLOCK)
    N, K = w.shape
    if N < 1 or K < 1:
        raise _lib.VitFp4Error(f"weight: at least one row and one column needed, got {tuple(w.shape)}")
    if bias is not None and (bias.shape != (N,) or bias.stride(0) != 1 and N > 1):
        raise _lib.VitFp4Error(f"bias: a contiguous ({N},) vector needed, got {tuple(bias.shape)}")


@torch.library.custom_op("vitfp4::cast_fp8_block", mutates_args=())
def cast_fp8_block_op(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.cast_fp8_block(x, block_rows)


@cast_fp8_block_op.register_fake
def _(x, block_rows):
    M, K = x.shape
    ldc, kb = (K + 15) // 16 * 16, (K + 127) // 128
    codes = x.new_empty((M, ldc), dtype=torch.float8_e4m3fn)[:, :K]
    if block_rows == 1:
        return codes, x.new_empty((kb, M), dtype=torch.float32).t()
    return codes, x.new_empty(((M + block_rows - 1) // block_rows, kb), dtype=torch.float32)


@torch.library.custom_op("vitfp4::gemm_fp8_block", mutates_args=())
def gemm_fp8_block_op(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                      bias: torch.Tensor | None, fp32_out: bool) -> torch.Tensor:
    return ops.gemm_fp8_block(a, a_scale, b, b_scale, bias, torch.float32 if fp32_out else torch.bfloat16)


@gemm_fp8_block_op.register_fake
def _(a, a_scale, b, b_scale, bias, fp32_out):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=torch.float32 if fp32_out else torch.bfloat16)


@torch.library.custom_op("vitfp4::linear_fp8_block", mutates_args=())
def linear_fp8_block_op(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                        bias: torch.Tensor | None) -> torch.Tensor:
    return ops.linear_fp8_block(x, w, w_scale, bias)


@linear_fp8_block_op.register_fake
def _(x, w, w_scale, bias):
    return x.new_empty((x.shape[0], w.shape[0]))


def _traced(*ts: torch.Tensor | None) -> bool:
    """Whether a call has to go through its torch.library op: under torch.compile or a dispatch mode (tracers, fake
    tensors), with tensors of a subclass, or where gradients are recorded (the op has no backward and says so).
    Plain calls skip the dispatcher, which costs more host time than the small kernels run."""
    if torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack():
        return True
    grad = torch.is_grad_enabled()
    for t in ts:
        if t is not None and (grad and t.requires_grad or type(t) not in _PLAIN):
            return True
    return False


def quantize_to_fp8_block(x: torch.Tensor, block_rows: int = 1):
    """(..., K) bf16 / fp32 -> (codes float8_e4m3fn (..., K), scale fp32 (..., ceil(K / 128))).

    ``block_rows`` 1: a scale per row and 128 columns (activations).  128: a scale per 128 x 128 block of a 2-D
    weight -> scale (ceil(N / 128), ceil(K / 128))."""
    if block_rows == 1 and not torch.compiler.is_compiling():
        out = ops.fast_cast(x)
        if out is not None:
            return out
    if block_rows not in (1, _BLOCK):
        raise _lib.VitFp4Error(f"block_rows is 1 or {_BLOCK}, got {block_rows}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise _lib.VitFp4Error(f"at least one column needed, got {tuple(x.shape)}")
    if x.dim() != 2 and block_rows != 1:
        raise _lib.VitFp4Error(f"a 2-D weight is needed for {_BLOCK} x {_BLOCK} blocks, got {tuple(x.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    codes, scale = (cast_fp8_block_op if _traced(x) else ops.cast_fp8_block)(x2, block_rows)
    if x.dim() == 2:
        return codes, scale
    return codes.unflatten(0, x.shape[:-1]) if x.dim() > 1 else codes[0], scale.reshape(*x.shape[:-1], scale.shape[-1])


def dequantize_fp8_block(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp32 values of an FP8 block operand (a small tensor utility, on whatever device its input lives on)."""
    K = codes.shape[-1]
    s = scale.repeat_interleave(_BLOCK, dim=-1)[..., :K]
    if s.shape[:-1] != codes.shape[:-1]:
        s = s.repeat_interleave(_BLOCK, dim=-2)[: codes.shape[-2]]
    return codes.float() * s


def fp8_block_gemm(a, a_scale, b, b_scale, *, bias=None, out_dtype=torch.bfloat16):
    """A (..., K) x B (N, K) in the FP8 block format -> (..., N) in bf16 or fp32, one rounding of the fp32 sum.

    ``a_scale`` (..., ceil(K / 128)), ``b_scale`` (ceil(N / 128), ceil(K / 128)), any strides; ``bias`` (N,) bf16 or
    fp32.  Codes whose rows do not start on 16-byte boundaries are copied first."""
    lead = a.shape[:-1]
    if len(lead) != 1:
        if a.dim() < 1 or a_scale.dim() < 1 or a_scale.shape[:-1] != lead or not a.shape[-1]:
            raise _lib.VitFp4Error(f"a: codes (..., K) and scales (..., ceil(K / 128)) needed, got {tuple(a.shape)} and "
                                   f"{tuple(a_scale.shape)}")
        a, a_scale = a.reshape(-1, a.shape[-1]), a_scale.reshape(lead.numel(), a_scale.shape[-1])
    _check_operand("a", a, a_scale, 1)
    _check_weight(b, b_scale, bias)
    if a.shape[1] != b.shape[1]:
        raise _lib.VitFp4Error(f"a and b differ in K: {tuple(a.shape)} and {tuple(b.shape)}")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise _lib.VitFp4Error(f"out_dtype is bf16 or fp32, got {out_dtype}")
    if _traced(a, a_scale, b, b_scale, bias):
        y = gemm_fp8_block_op(a, a_scale, b, b_scale, bias, out_dtype == torch.float32)
    else:
        y = ops.gemm_fp8_block(a, a_scale, b, b_scale, bias, out_dtype)
    return y if len(lead) == 1 else y.view(*lead, b.shape[0])


def fp8_block_linear(x, w, w_scale, *, bias=None):
    """Linear layer with an FP8 block weight: online cast of x (..., K), product, + bias; output in x.dtype."""
    if not torch.compiler.is_compiling():
        out = ops.fast_linear(x, w, w_scale, bias)
        if out is not None:
            return out
    _check_weight(w, w_scale, bias)
    if x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise _lib.VitFp4Error(f"x of shape {tuple(x.shape)} and a weight of {w.shape[1]} columns")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    y = (linear_fp8_block_op if _traced(x, w, w_scale, bias) else ops.linear_fp8_block)(x2, w, w_scale, bias)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], w.shape[0])
