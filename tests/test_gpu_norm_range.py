"""rms_norm and its gradient over rows of very different sizes: the reciprocal root's cube leaves f32's range long before
the root, the sums and the results do."""
import pytest
import torch

import mx_ref as ref
from gpu_util import banner

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
SUMS = 96 * 2.0 ** -24  # roundings of a norm (test_gpu_norm.py)


@pytest.fixture(scope="module")
def mlxq():
    import mlxq as m
    m.load()
    return m


def _randn(seed, shape, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _close(y, want, dtype, extra):
    tol = ref.UNIT[dtype] * want.abs() + extra * (1 + ref.UNIT[dtype]) + ref.TINY[dtype]
    assert y.dtype == dtype and y.shape == want.shape
    assert ((y.cpu().double() - want).abs() <= tol).all()


# Rows held in registers by a part of a wave, by one and by several waves, and rows that are read twice.
@pytest.mark.parametrize("dtype,D", [(BF16, 24), (F32, 96), (BF16, 515), (F32, 2050), (BF16, 16384), (F32, 8195), (BF16, 20001)])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_gradient_of_large_and_small_rows(mlxq, dtype, D, eps):
    """The same roundings as rows of size 1 have, at sizes from 1e-14 to 1e16 (with eps 0 the reciprocal root is up to 1e14)."""
    banner("rms_norm_backward", dtype, D, eps)
    size = torch.tensor([1e-14, 1e-13, 1e-10, 1e-3, 1.0, 1e5, 1e12, 1e13, 1e14, 1e15, 1e16], dtype=torch.float64)
    rows = len(size)
    x = (_randn(D, (rows, D), F32).double() * size[:, None]).to(dtype)
    dy, w = _randn(D + 1, (rows, D), dtype), (1 + 0.3 * _randn(7, (D,), F32)).to(dtype)
    eps32 = float(torch.tensor(eps, dtype=F32))
    for weight, dsum in ((w, None), (None, dy.flip(0))):
        dx, dw = mlxq.rms_norm_backward(dy.cuda(), x.cuda(), None if weight is None else weight.cuda(), None if dsum is None else dsum.cuda(), eps)
        want, want_w, mag, mag_w = ref.rms_norm_gradient(dy, x, weight, dsum, eps32)
        _close(dx, want, dtype, (3 * SUMS + 8 * 2.0 ** -24) * mag)
        if weight is not None:
            _close(dw, want_w, dtype, (SUMS + (rows + 96) * 2.0 ** -24) * mag_w)
    y = mlxq.rms_norm(x.cuda(), w.cuda(), eps=eps)
    want = ref.rms_norm(x, w, eps32)
    _close(y, want, dtype, SUMS * want.abs())
