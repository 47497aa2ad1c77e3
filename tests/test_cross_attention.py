"""cross_sdpa: refusals (no GPU)."""
import pytest
import torch

from vitfp4 import _lib
from vitfp4.nvfp4 import cross_sdpa

B16 = torch.bfloat16
Q, K = torch.zeros(2, 4, 3, 64, dtype=B16), torch.zeros(2, 2, 9, 64, dtype=B16)


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.VitFp4Error, match="CUDA"):
        cross_sdpa(Q, K, K)


@pytest.mark.parametrize("args,kw", [
    ((Q.float(), K, K), {}),
    ((Q, K.half(), K), {}),
    ((Q[0], K, K), {}),
    ((Q, K, K[:, :, :8]), {}),
    ((Q, K[:1], K[:1]), {}),
    ((Q[..., :32], K, K), {}),
    ((Q[:, :3], K, K), {}),
    ((Q, K[:, :0], K[:, :0]), {}),
    ((Q[..., :60], K[..., :60], K[..., :60]), {}),
    ((torch.zeros(2, 4, 3, 136, dtype=B16), torch.zeros(2, 2, 9, 136, dtype=B16), torch.zeros(2, 2, 9, 136, dtype=B16)), {}),
    ((Q, K, K), {"kv_lens": torch.zeros(3, dtype=torch.int32)}),
    ((Q, K, K), {"kv_lens": torch.zeros(2)}),
    ((Q, K, K), {"key_mask": torch.ones(2, 8, dtype=torch.bool)}),
    ((Q, K, K), {"key_mask": torch.ones(2, 9)}),
    ((Q, K, K), {"scale": float("nan")}),
    ((Q, K, K), {"scale": float("inf")}),
])
def test_arguments_are_checked(args, kw):
    with pytest.raises(_lib.VitFp4Error):
        cross_sdpa(*args, **kw)


def test_strides_of_single_entries_do_not_matter():
    from vitfp4.nvfp4 import ops
    one = torch.zeros(64, dtype=B16).as_strided((1, 2, 3, 8), (49, 24, 8, 1))       # one image, an odd batch stride
    assert ops._attn_view(one) is one and ops._attn_strides(one) == (0, 24, 8)
    head = torch.zeros(64, dtype=B16).as_strided((2, 1, 1, 8), (16, 3, 5, 1))
    assert ops._attn_view(head) is head and ops._attn_strides(head) == (16, 0, 0)
    two = torch.zeros(128, dtype=B16).as_strided((2, 2, 3, 8), (49, 24, 8, 1))
    copy = ops._attn_view(two)
    assert copy is not two and ops._attn_strides(copy) == (48, 24, 8)
