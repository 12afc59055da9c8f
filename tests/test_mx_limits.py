"""The decoder block's operators at the ends of their sizes, as far as the host decides on them (no GPU)."""
import ctypes

import pytest
import torch

import mlxq


@pytest.mark.parametrize("shape", [(4, 0, 64), (0, 3, 64), (2, 0, 3, 64), (2, 3, 0, 64)])
def test_no_heads_is_no_error_of_its_own(shape):
    """Tensors with an empty dimension get as far as any on the CPU do: to the wish for a GPU."""
    x = torch.empty(shape)
    for call in (lambda: mlxq.rms_norm(x), lambda: mlxq.rms_norm(x, torch.ones(64), x, mx=True), lambda: mlxq.rms_norm_backward(x, x, None, x)):
        with pytest.raises(ValueError, match="GPU tensors"):
            call()
    with pytest.raises((mlxq.MlxqError, ValueError), match="must be positive"):
        mlxq.rms_norm(torch.empty(*shape[:-1], 0))


def test_products_of_more_threads_than_a_launch_has():
    """Refused by name, before anything is launched: 2^30 features take 2^23 workgroups of 512."""
    from mlxq import _lib
    lib = _lib.load()
    at = 4096  # never read
    x, w = _lib.Mx(at, at, 4, _lib.MLXQ_MX_E4M3), _lib.Mx(at, at, 4, _lib.MLXQ_MX_E2M1)
    N = 2 ** 30 + 100
    assert lib.mlxq_mx_matmul(ctypes.byref(x), 1, 32, ctypes.byref(w), N, None, 0, at, 1, None) == _lib.MLXQ_EUNSUPPORTED
    assert "one launch" in lib.mlxq_last_error().decode()
    routing = _lib.Routed(at, at, at, at, 1, 1, 1)
    assert lib.mlxq_mx_experts(ctypes.byref(x), 0, 32, ctypes.byref(w), N, None, 0, ctypes.byref(routing), 0, at, 1, None, 0,
                               None) == _lib.MLXQ_EUNSUPPORTED
    assert "one launch" in lib.mlxq_last_error().decode()
