"""The decoder block's operators at the ends of their sizes, as far as the host decides on them (no GPU)."""
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
