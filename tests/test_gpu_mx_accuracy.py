"""What products of 8-bit rows lose where one product is much larger than its neighbours, as with features that stick out."""
import pytest
import torch

import mx_ref as ref
from gpu_util import banner

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mlxq():
    import mlxq as m
    m.load()
    return m


def _spiky(M, K):
    """Rows with one of eight neighbouring values 2^13 times the others and more, which the type just holds; alternating signs
    make every other row's large products cancel."""
    x = torch.full((M, K), 1.875 * 2.0 ** -6)
    x[:, ::8] = 256.0
    x[1::2, ::16] *= -1
    return x.to(torch.float8_e4m3fn), torch.full((M, -(-K // 128) * 4), 127, dtype=torch.uint8)[:, :K // 32]


def _weights(N, K, lead=()):
    """Codes of 1 (every third row with other codes and scales), two to a byte."""
    code = torch.full((*lead, N, K), 2, dtype=torch.long)
    code[..., 2::3, :] = torch.randint(1, 8, (K,), generator=torch.Generator().manual_seed(1))
    room = torch.full((*lead, N, -(-K // 128) * 4), 127, dtype=torch.uint8)
    room[..., 1::4, :] = 120
    return ref.packed(code, "e2m1"), room[..., :K // 32]


def _cuda(mlxq, mx):
    codes, scales = mx
    room = torch.zeros((*scales.shape[:-1], -(-scales.shape[-1] // 4) * 4), dtype=torch.uint8)
    room[..., :scales.shape[-1]] = scales
    return mlxq.Mx(codes.cuda(), room.cuda()[..., :scales.shape[-1]])


# one row, tiles of 16, 32, 64 and 128 rows, and K split over groups of waves
SHAPES = [(1, 32, 5), (1, 4096, 40), (3, 416, 6000), (20, 288, 17), (33, 2912, 640), (100, 160, 12001), (300, 1056, 520), (500, 160, 14002)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_spiky_rows_to_f16_and_f32(mlxq, M, K, N):
    """f32 sums and one rounding: nothing more than what 4-bit rows may be off by."""
    x, w = _spiky(M, K), _weights(N, K)
    xv, wv = ref.values(x), ref.values(w)
    want = xv @ wv.t()
    for dtype in (F32, F16):
        banner("mx_matmul", M, K, N, dtype)
        fits = want.abs() < torch.finfo(dtype).max
        assert fits.any()
        y = mlxq.mx_matmul(_cuda(mlxq, x), _cuda(mlxq, w), out_dtype=dtype).cpu().double()
        assert ((y - want).abs() <= ref.product_bound(xv, wv, dtype, "e2m1"))[fits].all()
        bias = -want[0].float()
        y = mlxq.mx_matmul(_cuda(mlxq, x), _cuda(mlxq, w), bias.cuda(), dtype).cpu().double()
        exact = want + bias.double()
        fits = exact.abs() < torch.finfo(dtype).max
        # f32 sums of the magnitudes and the bias's addition, then a rounding of what is left
        sums = ref.product_bound(xv, wv, F32, "e2m1") + 2.0 ** -23 * bias.double().abs()
        assert ((y - exact).abs() <= sums * (1 + ref.UNIT[dtype]) + ref.UNIT[dtype] * exact.abs() + ref.TINY[dtype])[fits].all()


@pytest.mark.parametrize("combine", [False, True])
def test_spiky_rows_through_experts(mlxq, combine):
    T, k, E, K, N = 60, 2, 4, 416, 70
    x, w = _spiky(T, K), _weights(N, K, (E,))
    ids = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).int()
    weights = torch.rand(T, k, generator=torch.Generator().manual_seed(3))
    routing = mlxq.route_plan(ids.cuda(), weights.cuda(), E)
    want, xv, wv = ref.experts(x, w, ids, None)
    tol = torch.stack([torch.stack([ref.product_bound(xv[t:t + 1], wv[e], F16, "e2m1")[0] for e in ids[t].tolist()]) for t in range(T)])
    y = mlxq.mx_experts(_cuda(mlxq, x), _cuda(mlxq, w), routing, combine=combine, out_dtype=F16).cpu().double()
    if combine:
        # products rounded to fp16, k weighted in f32 and rounded once
        mag = ((want.abs() + tol) * weights.double()[..., None]).sum(1)
        tol = (tol * weights.double()[..., None]).sum(1) + (k + 1) * 2.0 ** -23 * mag + ref.UNIT[F16] * mag + ref.TINY[F16]
        want = (want * weights.double()[..., None]).sum(1)
    # 65520 = 65504 + half a step and more round to infinity (two products of 36251 by weights of 0.92 and 0.94 come to 67446)
    over = want.abs() - tol >= 65520
    assert ((y - want).abs() <= tol)[want.abs() + tol < 65520].all() and torch.equal(y[over], want[over].sign() * float("inf"))


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_spiky_rows_to_bf16(mlxq, M, K, N):
    """The 8-bit instruction cuts each of eight neighbouring products below 2^-13 of the largest one: up to 7 2^-13 of it in all, less
    than half a rounding to bf16 of the magnitudes' sum."""
    x, w = _spiky(M, K), _weights(N, K)
    xv, wv = ref.values(x), ref.values(w)
    want = xv @ wv.t()
    lost = torch.zeros_like(want)
    for k in range(0, K, 8):  # weights of 1, or others of a row: the largest product is that of the largest value or a weight of 6
        p = xv[:2, None, k:k + 8].abs() * wv[None, :, k:k + 8].abs()
        lost += 7 * 2.0 ** -13 * p.amax(-1)[torch.arange(M) % 2]
    banner("mx_matmul", M, K, N)
    y = mlxq.mx_matmul(_cuda(mlxq, x), _cuda(mlxq, w), out_dtype=BF16).cpu().double()
    sums = ref.product_bound(xv, wv, F32, "e2m1") + lost
    assert (lost <= 2.0 ** -10 * (xv.abs() @ wv.abs().t())).all()
    assert ((y - want).abs() <= sums * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()).all()
