"""Dimensions of 2^31 and more are refused before they reach entry points that count in 32 bits (without a GPU: meta tensors hold nothing)."""
import pytest
import torch

import hipkittens_amd as hk
from hipkittens_amd import tk_kernel as tk

LONG = 2 ** 32 + 8   # 8 in its lower 32 bits


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_gated():
    with pytest.raises(RuntimeError, match="2\\^31"):
        tk.dispatch_gated_gemm(_meta(LONG, 8), _meta(16, 8), _meta(LONG, 8))
    with pytest.raises(RuntimeError, match="2\\^31"):
        tk.dispatch_gated_gemm(_meta(8, LONG), _meta(16, LONG), _meta(8, 8))
    with pytest.raises(RuntimeError, match="2\\^31"):
        tk.dispatch_gated_gemm_dgrad(_meta(LONG, 8), _meta(8, 8), _meta(LONG, 16), _meta(LONG, 16))


def test_products():
    with pytest.raises(RuntimeError, match="2\\^31"):
        tk.dispatch_bf16_gemm_dgrad(_meta(LONG, 8), _meta(8, 8), _meta(LONG, 8))
    with pytest.raises(RuntimeError, match="2\\^31"):
        tk.dispatch_bf16_gemm_wgrad(_meta(8, LONG), _meta(8, 8), _meta(LONG, 8))


def test_embedding():
    with pytest.raises(RuntimeError, match="2\\^31"):
        tk.dispatch_embedding(_meta(LONG, dtype=torch.int32), _meta(8, 8), _meta(LONG, 8))
    with pytest.raises(RuntimeError, match="2\\^31"):
        tk.dispatch_embedding_backward(_meta(8, dtype=torch.int64), _meta(8, 8), _meta(LONG, 8), _meta(64, dtype=torch.uint8))
    for shape in ((LONG, 8, 8), (8, LONG, 8), (8, 8, LONG)):
        assert hk.tk_kernel.embedding_backward_workspace_bytes(*shape) == 0
