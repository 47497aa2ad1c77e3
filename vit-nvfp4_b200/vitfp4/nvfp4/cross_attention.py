"""Cross attention: queries over an encoder's keys and values of another length.

The attention of pooling heads (one latent query per image), resamplers (tens of latents) and decoders over a
ViT's tokens, with shared key / value heads, a key count per image and a mask of keys.  bf16 operands, softmax and
accumulation in fp32, the weights rounded to bf16 for their product with the values (not for their sum, and not for
up to 4 rows over short keys), on the kernels of vf4_cross_attn.  No counterpart in the reference, whose attention is a
ViT's self attention (src/vit_nvfp4/nvfp4/attention.py:53-86).  Inference only: the op has no backward pass.
"""
from __future__ import annotations

import math

import torch

from .. import _lib
from . import ops
from .fp8_block import _traced


@torch.library.custom_op("vitfp4::cross_attention", mutates_args=())
def cross_attention_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, kv_lens: torch.Tensor | None,
                       key_mask: torch.Tensor | None) -> torch.Tensor:
    return ops.cross_attention(q, k, v, scale, kv_lens, key_mask)


@cross_attention_op.register_fake
def _(q, k, v, scale, kv_lens, key_mask):
    B, H, Sq, D = q.shape
    return q.new_empty((B, Sq, H, D)).transpose(1, 2)


def cross_sdpa(query, key, value, *, kv_lens=None, key_mask=None, scale=None):
    """softmax(scale * query key^T) value over the keys each image keeps -> (B, H, Sq, D) bf16.

    ``query`` (B, H, Sq, D), ``key`` and ``value`` (B, Hkv, Skv, D), all bf16, H a multiple of Hkv (query head h reads
    key head h // (H // Hkv)), D a multiple of 8 up to 128; any strides (views of packed projections and expanded
    tensors are read in place).  ``kv_lens`` (B,) int32 or int64: keys from kv_lens[b] on are not used.  ``key_mask``
    (B, Skv) bool: False keys are not used.  Unused keys and values may hold anything; a query without any used key
    gives 0, whatever it holds.  ``scale`` defaults to 1 / sqrt(D).  The result is laid out as (B, Sq, H, D), ready for the output
    projection."""
    if not torch.compiler.is_compiling():
        out = ops.fast_cross(query, key, value, kv_lens, key_mask, scale)
        if out is not None:
            return out
    for name, t in (("query", query), ("key", key), ("value", value)):
        if t.dtype != torch.bfloat16 or t.dim() != 4:
            raise _lib.VitFp4Error(f"{name}: a 4-D bf16 tensor needed, got {tuple(t.shape)} {t.dtype}")
    B, H, _, D = query.shape
    if key.shape != value.shape or key.shape[0] != B or key.shape[3] != D:
        raise _lib.VitFp4Error(f"key and value of one shape (B, Hkv, Skv, D) with query's B and D needed, got "
                               f"{tuple(query.shape)}, {tuple(key.shape)}, {tuple(value.shape)}")
    Hkv, Skv = key.shape[1], key.shape[2]
    if Hkv < 1 or H < 1 or H % Hkv:
        raise _lib.VitFp4Error(f"{H} query heads are no multiple of {Hkv} key heads")
    if D % 8 or not 8 <= D <= 128:
        raise _lib.VitFp4Error(f"head dims that are multiples of 8 up to 128, got {D}")
    if kv_lens is not None:
        if tuple(kv_lens.shape) != (B,) or kv_lens.dtype not in (torch.int32, torch.int64):
            raise _lib.VitFp4Error(f"kv_lens: ({B},) int32 or int64 needed, got {tuple(kv_lens.shape)} {kv_lens.dtype}")
        if kv_lens.dtype != torch.int32:
            kv_lens = kv_lens.clamp(0, Skv).to(torch.int32)
        elif not kv_lens.is_contiguous():
            kv_lens = kv_lens.contiguous()
    if key_mask is not None:
        if tuple(key_mask.shape) != (B, Skv) or key_mask.dtype != torch.bool:
            raise _lib.VitFp4Error(f"key_mask: ({B}, {Skv}) bool needed, got {tuple(key_mask.shape)} {key_mask.dtype}")
        if key_mask.stride(1) != 1 and Skv > 1:
            key_mask = key_mask.contiguous()
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise _lib.VitFp4Error(f"scale is not finite: {scale}")
    if _traced(query, key, value, kv_lens, key_mask):
        return cross_attention_op(query, key, value, scale, kv_lens, key_mask)
    return ops.cross_attention(query, key, value, scale, kv_lens, key_mask)
