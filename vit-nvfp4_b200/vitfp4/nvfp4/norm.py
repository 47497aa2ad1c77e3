"""Norms before and after a block, fused with the block's gate and residual scale.

    x' = x + residual_scale * gate * N_post(y),    h = N_pre(x')

The step between two blocks of a sandwich-norm or adaLN-gated transformer; a timm / DINOv2 block's
``x + ls(y); norm(x)`` is the case without a post-norm and with LayerScale as the gate (the NVFP4 path has its own
form of that one, with the NVFP4 cast: ``ops.ln_cast``).  No counterpart kernel in the reference, which leaves norms
to eager torch or torch.compile.  Inference only: the op has no backward pass.
"""
from __future__ import annotations

import torch

from .. import _lib
from . import ops
from .fp8_block import _traced

_OptT = torch.Tensor | None


@torch.library.custom_op("vitfp4::gated_residual_norm", mutates_args=())
def gated_residual_norm_op(x: torch.Tensor, y: torch.Tensor | None, gate: torch.Tensor | None, residual_scale: float,
                           post: str, post_w: torch.Tensor | None, post_b: torch.Tensor | None, pre: str,
                           pre_w: torch.Tensor | None, pre_b: torch.Tensor | None, eps: float,
                           fp8_out: bool) -> list[torch.Tensor]:
    out = ops.gated_residual_norm(x, y, gate, residual_scale, post or None, post_w, post_b, pre or None, pre_w, pre_b,
                                  eps, fp8_out)
    return [t for t in out if t is not None]


@gated_residual_norm_op.register_fake
def _(x, y, gate, residual_scale, post, post_w, post_b, pre, pre_w, pre_b, eps, fp8_out):
    M, K = x.shape
    out = [] if y is None else [x.new_empty((M, K))]
    if pre and fp8_out:
        out += [x.new_empty((M, (K + 15) // 16 * 16), dtype=torch.float8_e4m3fn)[:, :K],
                x.new_empty(((K + 127) // 128, M), dtype=torch.float32).t()]
    elif pre:
        out.append(x.new_empty((M, K)))
    return out


def _check_param(name: str, t: _OptT, K: int) -> None:
    if t is not None and (tuple(t.shape) != (K,) or t.stride(0) != 1 and K > 1):
        raise _lib.VitFp4Error(f"{name}: a contiguous ({K},) vector needed, got {tuple(t.shape)}")


def gated_residual_norm(x, y, *, gate=None, residual_scale=1.0, norm="layer", post_norm=True, post_weight=None,
                        post_bias=None, pre_norm=True, pre_weight=None, pre_bias=None, eps=1e-6, out_dtype=None):
    """(x', h) of x (..., K) and y (..., K) bf16 / fp32: x' = x + residual_scale * gate * N_post(y), h = N_pre(x').

    ``norm`` is "layer" or "rms"; ``post_norm`` / ``pre_norm`` False leave that norm out (h is then None without a
    pre-norm).  ``gate`` is (K,), or (G, K) with the rows divided into G equal runs (a gate per image).
    ``out_dtype`` None or x's: h in x's type; ``torch.float8_e4m3fn``: h = (codes, scales) in the FP8 block format
    that ``fp8_block_gemm`` reads, those that ``quantize_to_fp8_block`` gives for the fp32 values.  ``y`` None: (x, N_pre(x)).  Arithmetic in fp32; x' is rounded once for storage
    and enters N_pre unrounded."""
    if post_norm and pre_norm and norm in ops.NORM_KINDS and not torch.compiler.is_compiling() and \
            (out_dtype is None or out_dtype == torch.float8_e4m3fn):
        out = ops.fast_norm(x, y, gate, residual_scale, ops.NORM_KINDS[norm], post_weight, post_bias, pre_weight,
                            pre_bias, eps, out_dtype is not None)
        if out is not None:
            return out
    if norm not in ("layer", "rms"):
        raise _lib.VitFp4Error(f"norm is 'layer' or 'rms', got {norm!r}")
    if x.dtype not in (torch.bfloat16, torch.float32) or x.dim() < 1 or x.shape[-1] < 1:
        raise _lib.VitFp4Error(f"x: (..., K) bf16 or fp32 needed, got {tuple(x.shape)} {x.dtype}")
    K = x.shape[-1]
    if y is None:
        if gate is not None or post_weight is not None or post_bias is not None or not pre_norm:
            raise _lib.VitFp4Error("without y there is only the pre-norm")
        post_norm = False
    elif y.shape != x.shape or y.dtype != x.dtype:
        raise _lib.VitFp4Error(f"y: x's shape and type needed ({tuple(x.shape)} {x.dtype}), got {tuple(y.shape)} {y.dtype}")
    if not post_norm and (post_weight is not None or post_bias is not None):
        raise _lib.VitFp4Error("a post-norm weight or bias without the post-norm")
    if not pre_norm and (pre_weight is not None or pre_bias is not None or out_dtype not in (None, x.dtype)):
        raise _lib.VitFp4Error("a pre-norm weight, bias or output type without the pre-norm")
    if out_dtype not in (None, x.dtype, torch.float8_e4m3fn):
        raise _lib.VitFp4Error(f"out_dtype is {x.dtype} or float8_e4m3fn, got {out_dtype}")
    M = x.numel() // K
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.shape[-1] != K or not gate.is_contiguous():
            raise _lib.VitFp4Error(f"gate: a contiguous ({K},) or (G, {K}) tensor needed, got {tuple(gate.shape)}")
        if gate.dim() == 2 and (gate.shape[0] < 1 or M % gate.shape[0]):
            raise _lib.VitFp4Error(f"{M} rows do not divide into {gate.shape[0]} gates")
    _check_param("post_weight", post_weight, K)
    _check_param("post_bias", post_bias, K)
    _check_param("pre_weight", pre_weight, K)
    _check_param("pre_bias", pre_bias, K)
    params = (gate, post_weight, post_bias, pre_weight, pre_bias)
    dtypes = {t.dtype for t in params if t is not None}
    if dtypes and dtypes != {x.dtype} and dtypes != {torch.float32}:
        if not dtypes <= {torch.bfloat16, torch.float32, torch.float16}:
            raise _lib.VitFp4Error(f"gate, weights and biases are bf16 or fp32, got {sorted(map(str, dtypes))}")
        params = [None if t is None else t.float() for t in params]   # fp32 holds every bf16 and fp16 value
    fp8 = out_dtype == torch.float8_e4m3fn
    x2, y2 = (t if t is None or t.dim() == 2 else t.reshape(-1, K) for t in (x, y))
    gate, *rest = params
    kind = (norm if post_norm else None, norm if pre_norm else None)
    if _traced(x, y, *params):
        out = gated_residual_norm_op(x2, y2, gate, float(residual_scale), kind[0] or "", rest[0], rest[1], kind[1] or "",
                                     rest[2], rest[3], float(eps), fp8)
        out = list(out)
        new = x2 if y is None else out.pop(0)
        h, scale = out if fp8 else (out[0] if out else None, None)
    else:
        new, h, scale = ops.gated_residual_norm(x2, y2, gate, residual_scale, kind[0], rest[0], rest[1], kind[1], rest[2],
                                                rest[3], eps, fp8)
    new = x if y is None else new if x.dim() == 2 else new.view(x.shape)
    if h is not None and x.dim() != 2:
        h = h.unflatten(0, x.shape[:-1]) if x.dim() > 1 else h[0]
        scale = None if scale is None else scale.reshape(*x.shape[:-1], scale.shape[-1])
    return new, ((h, scale) if fp8 else h)
