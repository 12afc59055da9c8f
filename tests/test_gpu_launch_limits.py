"""Casts and epilogues of 2^32 elements and more, a thread each: a launch counts its threads in 32 bits, and of more of them it runs
a part without an error."""
import pytest
import torch

from gpu_util import banner

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def mlxq():
    import mlxq as m
    m.load()
    return m


def _fill(n, dtype):
    """Memory that the next tensor of this size gets, full of NaN."""
    t = torch.full((n,), float("nan"), dtype=dtype, device="cuda")
    del t


def test_cast(mlxq):
    from mlxq import _lib
    n = 2 ** 32 + 1000
    x = torch.empty(n, dtype=BF16, device="cuda")
    for k in range(0, n, 2 ** 28):
        x[k:k + 2 ** 28] = torch.arange(k, min(k + 2 ** 28, n), device="cuda") % 251
    y = torch.full((n,), float("nan"), dtype=F32, device="cuda")
    banner("cast", n)
    lib = _lib.load()
    _lib.check(lib.mlxq_cast(x.data_ptr(), _lib.MLXQ_BFLOAT16, y.data_ptr(), _lib.MLXQ_FLOAT32, n, torch.cuda.current_stream().cuda_stream))
    for k in range(0, n, 2 ** 28):
        assert torch.equal(y[k:k + 2 ** 28], x[k:k + 2 ** 28].float())
    x.fill_(float("nan"))
    _lib.check(lib.mlxq_cast(y.data_ptr(), _lib.MLXQ_FLOAT32, x.data_ptr(), _lib.MLXQ_BFLOAT16, n, torch.cuda.current_stream().cuda_stream))
    for k in range(0, n, 2 ** 28):
        assert torch.equal(x[k:k + 2 ** 28].float(), y[k:k + 2 ** 28])


def test_promoted_linear(mlxq):
    """bf16 rows and an f32 bias: the product is widened by the elementwise epilogue."""
    M, K, N = 2 ** 20 + 300, 64, 4100
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(M, K, generator=g, device="cuda").to(BF16)
    wq, s, b = mlxq.quantize((torch.randn(N, K, generator=g, device="cuda") / 8).to(BF16), 64, 4)
    bias = torch.randn(N, generator=g, device="cuda")
    banner("linear", M, K, N)
    _fill(M * N, F32)
    y = mlxq.linear(x, wq, s, b, 64, 4, bias=bias)
    assert y.dtype == F32 and y.shape == (M, N) and M * N > 2 ** 32
    w = mlxq.dequantize(wq, s, b, 64, 4).double().cpu()
    border = 16777215 * 256 // N
    for rows in (slice(0, 20), slice(border - 20, border + 20), slice(M - 20, M)):
        p = x[rows].cpu().double() @ w.t()
        # the product's f32 sums of 64 terms, its rounding to bf16, and the f32 addition of the bias
        mag = x[rows].cpu().double().abs() @ w.abs().t()
        tol = 2.0 ** -8 * p.abs() + 70 * 2.0 ** -24 * mag * (1 + 2.0 ** -8) + 2.0 ** -24 * (p.abs() + bias.cpu().double().abs()) * (1 + 2.0 ** -6)
        assert ((y[rows].cpu().double() - (p + bias.cpu().double())).abs() <= tol).all()
    for k in range(0, M, 2 ** 17):
        assert bool(y[k:k + 2 ** 17].isfinite().all())
