"""gated_residual_norm: refusals (no GPU)."""
import pytest
import torch

from vitfp4 import _lib
from vitfp4.nvfp4 import gated_residual_norm

X = torch.zeros(6, 32)


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.VitFp4Error, match="CUDA"):
        gated_residual_norm(X, X)


@pytest.mark.parametrize("args,kw", [
    ((X, X), {"norm": "batch"}),
    ((X.half(), X.half()), {}),
    ((X, X[:3]), {}),
    ((X, X.bfloat16()), {}),
    ((X, None), {"gate": torch.ones(32)}),
    ((X, None), {"post_weight": torch.ones(32)}),
    ((X, None), {"pre_norm": False}),
    ((X, X), {"post_norm": False, "post_bias": torch.ones(32)}),
    ((X, X), {"pre_norm": False, "pre_weight": torch.ones(32)}),
    ((X, X), {"pre_norm": False, "out_dtype": torch.float8_e4m3fn}),
    ((X, X), {"out_dtype": torch.float16}),
    ((X, X), {"gate": torch.ones(31)}),
    ((X, X), {"gate": torch.ones(4, 32)}),
    ((X, X), {"gate": torch.ones(32, 2).t()}),
    ((X, X), {"pre_weight": torch.ones(33)}),
    ((X, X), {"pre_weight": torch.ones(64)[::2]}),
    ((X, X), {"pre_weight": torch.ones(32, dtype=torch.int32)}),
])
def test_arguments_are_checked(args, kw):
    with pytest.raises(_lib.VitFp4Error):
        gated_residual_norm(*args, **kw)
