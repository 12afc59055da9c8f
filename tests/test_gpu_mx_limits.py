"""The decoder block's operators at the ends of their sizes: nothing to do, more rows than one launch has threads for, and what
lies beside their results."""
import ctypes

import pytest
import torch

import mx_ref as ref
from gpu_util import banner

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def mlxq():
    import mlxq as m
    m.load()
    return m


@pytest.mark.parametrize("shape", [(4, 0, 64), (0, 3, 64), (2, 0, 3, 64), (2, 3, 0, 64), (0, 0, 32)])
def test_no_heads(mlxq, shape):
    """Any dimension but the last may be empty."""
    x, w = torch.empty(shape, device="cuda", dtype=BF16), torch.ones(shape[-1], device="cuda", dtype=BF16)
    y, h = mlxq.rms_norm(x, w, x)
    assert y.shape == h.shape == mlxq.rms_norm(x, w).shape == shape
    q = mlxq.rms_norm(x, w, mx=True)
    assert q.codes.shape == shape and q.scales.shape == (*shape[:-1], shape[-1] // 32)
    dx, dw = mlxq.rms_norm_backward(x, x, w, x)
    assert dx.shape == shape and dw.shape == w.shape and not dw.any()
    assert mlxq.mx_dequantize(mlxq.mx_quantize(x)).shape == shape
    few = mlxq.mx_quantize(torch.randn(5, shape[-1], device="cuda"))
    assert mlxq.mx_matmul(mlxq.mx_quantize(x, "e4m3"), few).shape == (*shape[:-1], 5)
