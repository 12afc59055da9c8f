"""Sizes that take more threads than a launch has, 2^32: refused before anything is launched, where they are not launched in parts.
(A launch of more runs a part of them, without an error.)  No GPU: the addresses are never followed."""
import ctypes

import pytest

from mlxq import _lib

P = 4096
BF16 = _lib.MLXQ_BFLOAT16


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _large(lib, status):
    assert status == _lib.MLXQ_EINVAL
    msg = lib.mlxq_last_error().decode()
    assert "too large" in msg or "too many" in msg, msg


def test_elementwise_calls(lib):
    n = 2 ** 32  # threads, each of 32, 8 or 8 values
    _large(lib, lib.mlxq_quantize(P, BF16, n, 32, 32, 4, P, P, P, None))
    _large(lib, lib.mlxq_dequantize(P, P, P, BF16, n // 4, 32, 32, 4, P, None))
    _large(lib, lib.mlxq_embedding(P, n // 4, P, P, P, BF16, 100, 32, 32, 4, P, BF16, None))


def test_products(lib):
    N = 2 ** 21
    for M, sb in ((2 ** 20, BF16), (2 ** 20, _lib.MLXQ_FLOAT32)):
        _large(lib, lib.mlxq_quantized_matmul(P, BF16, M * 128, 64, P, P, P, sb, N, 1, 64, 4, P, None))
    _large(lib, lib.mlxq_qmv_valu(P, _lib.MLXQ_FLOAT32, 1, 64, P, P, P, _lib.MLXQ_FLOAT32, 2 ** 28 + 16, 64, 4, P, None))


def test_serving_calls(lib):
    freqs = (ctypes.c_double * 64)(*[1.0] * 64)
    _large(lib, lib.mlxq_rotary_table(freqs, 64, 1.0, 2 ** 27, P, None))
    _large(lib, lib.mlxq_cache_copy_pages(P, 2 ** 12, 2 ** 24, 2 ** 20, 16, 16, P, P, 2 ** 13, None, 0, 0, 0, None))
