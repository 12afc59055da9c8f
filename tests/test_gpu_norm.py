"""rms_norm and rms_norm_backward against their definitions (mx_ref), on the GPU."""
import ctypes

import pytest
import torch

import mx_ref as ref
from gpu_util import banner

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# A row's f32 sum adds up at most 64 values a lane, 6 steps in a wave and 16 waves; then a division, a root, a reciprocal and
# two products: fewer than 96 roundings, each off by 2^-24.
SUMS = 96 * 2.0 ** -24


@pytest.fixture(scope="module")
def mlxq():
    import mlxq as m
    m.load()
    return m


def _x(seed, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _close(y, want, dtype, rel=SUMS, extra=0.0):
    tol = (rel + ref.UNIT[dtype]) * want.abs() + extra * (1 + ref.UNIT[dtype]) + ref.TINY[dtype]
    assert y.dtype == dtype and y.shape == want.shape
    assert ((y.cpu().double() - want).abs() <= tol).all()


DIMS = [1, 2, 3, 5, 7, 8, 31, 64, 65, 80, 127, 128, 255, 256, 257, 500, 513, 1023, 1024, 1025, 2047, 2050, 4096, 5000, 8191, 8192, 16384, 16391, 32768]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", DIMS)
def test_norm(mlxq, dtype, D):
    for rows, w_dtype, residual in ((1, None, False), (5, dtype, True), (33, F32, True), (3, BF16, False)):
        banner("rms_norm", dtype, D, rows, w_dtype, residual)
        x, r = _x(D, (rows, D), dtype, 2.0), _x(D + 1, (rows, D), dtype)
        w = None if w_dtype is None else (1 + 0.3 * _x(7, (D,), F32)).to(w_dtype)
        out = mlxq.rms_norm(x.cuda(), None if w is None else w.cuda(), r.cuda() if residual else None, 1e-5)
        y = out
        if residual:
            y, h = out
            x = (x.float() + r.float()).to(dtype)
            assert torch.equal(h.cpu(), x)
        _close(y, ref.rms_norm(x, w, 1e-5), dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 256, 512, 1056, 4096, 5120, 8224, 16384, 32768])
def test_norm_to_8_bits(mlxq, dtype, D):
    """Codes and scales are those of the exact norm: rounded from 64 bits, whatever the order of the sum."""
    for rows, residual in ((1, False), (6, True), (70, True)):
        banner("rms_norm mx", dtype, D, rows, residual)
        x, r, w = _x(D, (rows, D), dtype, 2.0), _x(D + 1, (rows, D), dtype), (1 + 0.3 * _x(7, (D,), F32)).to(dtype)
        out = mlxq.rms_norm(x.cuda(), w.cuda(), r.cuda() if residual else None, 1e-5, mx=True)
        q = out
        if residual:
            q, h = out
            x = (x.float() + r.float()).to(dtype)
            assert torch.equal(h.cpu(), x)
        code, scale = ref.quantized(ref.rms_norm(x, w, float(torch.tensor(1e-5))), "e4m3")
        assert torch.equal(ref.unpacked(q.codes), code) and torch.equal(q.scales.cpu().long(), scale)


def test_norm_of_extremes(mlxq):
    """Rows of zeros, of tiny and of large values, with infinities and NaN: each row by itself."""
    x = _x(1, (7, 96), F32)
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e15
    x[3, 5], x[4, 6] = float("inf"), float("nan")
    x[5, :] = 0
    x[5, 95] = 3.0
    y = mlxq.rms_norm(x.cuda(), None, eps=1e-6).cpu()
    want = ref.rms_norm(x, None, 1e-6)
    for row in (0, 1, 2, 5, 6):
        assert ((y[row].double() - want[row]).abs() <= (SUMS + 2.0 ** -24) * want[row].abs() + 2.0 ** -140).all()
    assert y[4].isnan().all() and torch.equal(y[3].isnan(), want[3].isnan()) and y[3].nan_to_num().abs().max() == 0
    q = mlxq.rms_norm(x.cuda(), None, eps=1e-6, mx=True)
    scales = q.scales.cpu().long()
    assert (scales[4] == 255).all() and (scales[3, 0] == 255) and (scales[3, 1:] != 255).all()
    assert (scales[0] == 0).all() and not ref.unpacked(q.codes)[0].any()


def test_norm_strides(mlxq):
    """Heads sliced from a projection, odd offsets, transposed and broadcast rows, leading dimensions; both call paths."""
    base = _x(3, (12, 11, 160), BF16).cuda()
    odd = _x(4, (40, 171), F32).cuda()
    w = (1 + 0.1 * _x(5, (160,), F32)).cuda()
    for x, weight in ((base[:, 2:7], w), (base[:, 3], w), (base[::2, ::3], w), (base.transpose(0, 1), w), (base[:, :, 3:100], None),
                      (odd[:, 1:], None), (odd.t(), None), (odd[:1].expand(9, 171), None), (base[0, 0], w),
                      (base.view(3, 4, 11, 160)[:, 1:3], w), (base.view(3, 4, 11, 160).permute(2, 0, 1, 3), w), (base[:, :1].expand(12, 5, 160), w)):
        for residual in (None, x.flip(0).contiguous(), x):
            got = mlxq.rms_norm(x, weight, residual)
            y, h = got if residual is not None else (got, x)
            want_h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
            assert torch.equal(h, want_h) and y.shape == x.shape
            _close(y, ref.rms_norm(want_h.cpu(), None if weight is None else weight.cpu(), 1e-6), x.dtype)


def test_norm_writes_its_rows_only(mlxq):
    """In place through the C interface, with rows apart: what lies between them stays."""
    from mlxq import _lib
    for D in (5, 64, 77, 2048):
        buf = torch.full((6, D + 9), 5.0, device="cuda", dtype=BF16)
        x = _x(D, (6, D), BF16).cuda()
        buf[:, :D] = x
        v = _lib.Heads(buf.data_ptr(), 1, D + 9, 0)
        _lib.check(_lib.load().mlxq_rms_norm(ctypes.byref(v), 1, 6, D, None, None, None, 0, 1e-6, ctypes.byref(v), None,
                                             torch.cuda.current_stream().cuda_stream))
        _close(buf[:, :D], ref.rms_norm(x.cpu(), None, 1e-6), BF16)
        assert (buf[:, D:] == 5).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", DIMS)
def test_gradient(mlxq, dtype, D):
    for rows, w_dtype, dsum in ((1, None, True), (5, dtype, False), (70, F32, True), (1100 if D < 600 else 40, dtype, True)):
        banner("rms_norm_backward", dtype, D, rows, w_dtype, dsum)
        x, dy, ds = _x(D, (rows, D), dtype, 2.0), _x(D + 1, (rows, D), dtype), _x(D + 2, (rows, D), dtype) if dsum else None
        w = None if w_dtype is None else (1 + 0.3 * _x(7, (D,), F32)).to(w_dtype)
        dx, dw = mlxq.rms_norm_backward(dy.cuda(), x.cuda(), None if w is None else w.cuda(), None if ds is None else ds.cuda(), 1e-5)
        want, want_w, mag, mag_w = ref.rms_norm_gradient(dy, x, w, ds, 1e-5)
        # r enters three times and the sum of g x once: three times the roundings of a norm, and a few more
        _close(dx, want, dtype, 0.0, (3 * SUMS + 8 * 2.0 ** -24) * mag)
        if w is None:
            assert dw is None
        else:
            # a term has the roundings of a norm; a workgroup adds up its rows, then at most 64 parts follow one another and 16 more
            _close(dw, want_w, w_dtype, 0.0, (SUMS + (rows + 96) * 2.0 ** -24) * mag_w)


def test_gradient_strides_and_heads(mlxq):
    base = [_x(s, (50, 9, 96), BF16).cuda() for s in range(3)]
    w = (1 + 0.1 * _x(5, (96,), F32)).to(BF16).cuda()
    for cut in (lambda t: t[:, 2:8], lambda t: t[::3], lambda t: t.transpose(0, 1), lambda t: t[:, 0], lambda t: t[:, 1:4, 5:90],
                lambda t: t.view(5, 10, 9, 96).permute(2, 0, 1, 3)):
        dy, x, ds = (cut(t) for t in base)
        weight = w[:x.shape[-1]].contiguous()
        dx, dw = mlxq.rms_norm_backward(dy, x, weight, ds)
        want, want_w, mag, mag_w = ref.rms_norm_gradient(dy.cpu(), x.cpu(), weight.cpu(), ds.cpu(), 1e-6)
        _close(dx, want, BF16, 0.0, (3 * SUMS + 8 * 2.0 ** -24) * mag)
        _close(dw, want_w, BF16, 0.0, (SUMS + 550 * 2.0 ** -24) * mag_w)


def test_gradient_is_that_of_differences(mlxq):
    """Central differences of the definition in 64 bits, at h = 2^-12: their own error is h^2 / 6 times a third derivative, which
    is below 64 sum |g| r^3 here (x of about 1, r of about 1), and 2^-50 of the function over h."""
    D, eps, h = 24, 1e-5, 2.0 ** -12
    x, dy, ds, w = _x(1, (3, D), F32), _x(2, (3, D), F32), _x(3, (3, D), F32), 1 + 0.3 * _x(4, (D,), F32)
    dx, dw = (t.cpu().double() for t in mlxq.rms_norm_backward(dy.cuda(), x.cuda(), w.cuda(), ds.cuda(), eps))
    f = lambda x, w: (ref.rms_norm(x, w, eps) * dy.double()).sum() + (x.double() * ds.double()).sum()  # noqa: E731
    _, _, mag, mag_w = ref.rms_norm_gradient(dy, x, w, ds, eps)
    slack = h * h / 6 * 64 * (dy.double() * w.double()).abs().sum() + 2.0 ** -50 * 100 / h
    for r in range(3):
        for e in range(0, D, 5):
            up, dn = x.double().clone(), x.double().clone()
            up[r, e] += h
            dn[r, e] -= h
            assert abs(float(dx[r, e] - (f(up, w) - f(dn, w)) / (2 * h))) <= float(mag[r, e]) * 300 * 2.0 ** -24 + float(slack)
    for e in range(0, D, 7):
        up, dn = w.double().clone(), w.double().clone()
        up[e] += h
        dn[e] -= h
        assert abs(float(dw[e] - (f(x, up) - f(x, dn)) / (2 * h))) <= float(mag_w[e]) * 200 * 2.0 ** -24 + 2.0 ** -50 * 100 / h


@pytest.mark.parametrize("dtype,D", [(BF16, 515), (F32, 1026), (BF16, 5121), (F16, 16399), (BF16, 24580), (F32, 8195), (F32, 20001)])
def test_gradient_in_place(mlxq, dtype, D):
    """dx over dy, and over dsum, with rows that end inside a piece and a buffer that goes on behind them: the same bits."""
    x, dy, ds = (_x(D + i, (300, D), dtype).cuda() for i in range(3))
    w = (1 + 0.3 * _x(7, (D,), F32)).to(dtype).cuda()
    want, want_w = mlxq.rms_norm_backward(dy, x, w, ds, 1e-5)
    lib, code = mlxq._lib.load(), mlxq.mx._dt(x)
    need = lib.mlxq_rms_norm_backward_workspace_size(300, 1, D, code)
    ws, dw = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda"), torch.empty_like(w)
    view = lambda t: ctypes.byref(mlxq._lib.Heads(t.data_ptr(), 1, t.stride(0), 0))  # noqa: E731
    for over in (0, 1):
        bufs = [torch.full((300, D + 7), 5.0, dtype=dtype, device="cuda") for _ in range(2)]
        bufs[0][:, :D], bufs[1][:, :D] = dy, ds
        mlxq._lib.check(lib.mlxq_rms_norm_backward(view(bufs[0]), view(x), code, 300, D, w.data_ptr(), code, view(bufs[1]), 1e-5,
                                                   view(bufs[over]), dw.data_ptr(), ws.data_ptr(), need,
                                                   torch.cuda.current_stream().cuda_stream))
        assert torch.equal(bufs[over][:, :D], want) and torch.equal(dw, want_w) and (bufs[over][:, D:] == 5).all()


def test_gradient_bits_repeat(mlxq):
    x, dy, w = (_x(s, (5000, 1000), BF16).cuda() for s in (1, 2, 3))
    w = w[0].contiguous()
    first = mlxq.rms_norm_backward(dy, x, w)
    for _ in range(4):
        again = mlxq.rms_norm_backward(dy, x, w)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_empty(mlxq):
    x, w = torch.empty(0, 64, device="cuda", dtype=BF16), torch.ones(64, device="cuda", dtype=BF16)
    assert mlxq.rms_norm(x, w).shape == (0, 64) and mlxq.rms_norm(x, w, mx=True).codes.shape == (0, 64)
    y, h = mlxq.rms_norm(x, w, x)
    assert y.shape == h.shape == (0, 64)
    dx, dw = mlxq.rms_norm_backward(x, x, w)
    assert dx.shape == (0, 64) and not dw.any() and dw.shape == (64,)


def test_past_32_bits(mlxq):
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(70000, 32768, generator=g, device="cuda", dtype=BF16)  # 4.6 GB
    w = torch.ones(32768, device="cuda", dtype=BF16)
    y = mlxq.rms_norm(x, w)
    dx, _ = mlxq.rms_norm_backward(x, x, w)
    for r in (0, 65600, 69999):
        _close(y[r], ref.rms_norm(x[r].cpu(), None, 1e-6), BF16)
        want, _, mag, _ = ref.rms_norm_gradient(x[r:r + 1].cpu(), x[r:r + 1].cpu(), None, None, 1e-6)
        _close(dx[r:r + 1], want, BF16, 0.0, (3 * SUMS + 8 * 2.0 ** -24) * mag)
