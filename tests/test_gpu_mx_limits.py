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


def test_norm_of_more_rows_than_a_launch_has_threads_for(mlxq):
    """2^29 rows of 8 lanes are 2^32 threads: rows at both ends and around the border."""
    rows = 2 ** 29 + 1000
    x = torch.randn(rows, 1, device="cuda", generator=torch.Generator("cuda").manual_seed(1), dtype=BF16)
    banner("rms_norm", rows)
    y = torch.empty_like(x)
    for part in range(2):  # y holds what no norm gives, so that rows left out show
        y.fill_(7.0)
        del y
        y = mlxq.rms_norm(x)
    border = 16777215 * 32
    for a, b in ((0, 1000), (border - 1000, border + 1000), (2 ** 29 - 1000, 2 ** 29), (rows - 1000, rows)):
        want = ref.rms_norm(x[a:b].cpu(), None, 1e-6)
        assert ((y[a:b].cpu().double() - want).abs() <= (96 * 2.0 ** -24 + 2.0 ** -8) * want.abs() + 2.0 ** -134).all()
    # every row: signs survive, and no magnitude passes 1
    assert bool((torch.sign(y) == torch.sign(x)).all()) and bool((y.abs() <= 1).all())


def test_routing_of_more_tokens_than_a_launch_has_threads_for(mlxq):
    """2^26 tokens, a wave each."""
    T, E = 2 ** 26 + 9, 4
    z = torch.randn(T, E, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    active = torch.ones(T, dtype=torch.bool, device="cuda")
    active[-3], active[5] = False, False
    banner("route_experts", T, E)
    r = mlxq.route_experts(z, 1, normalize=False, active=active)
    none = r.ids[:, 0] < 0
    assert torch.equal(none, ~active)
    top = z.amax(-1)
    at = torch.where(none, 0, r.ids[:, 0]).long()
    assert bool(((z.gather(1, at[:, None])[:, 0] == top) | none).all())
    counts = torch.stack([(r.ids == e).sum() for e in range(E)])
    assert torch.equal(r.starts.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))
    key = torch.where(none, E, r.ids[:, 0])[r.rows.long()]
    assert bool((key[1:] >= key[:-1]).all()) and bool(((r.rows[1:] > r.rows[:-1]) | (key[1:] > key[:-1])).all())
    del key, at, top
    dw = torch.randn(T, 1, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    dz = mlxq.route_experts_backward(dw, z, r.ids, normalize=False)
    border = 16777215 * 4
    for a, b in ((0, 100), (border - 100, border + 100), (T - 200, T)):
        zc, ids = z[a:b].cpu(), r.ids[a:b].cpu()
        want, w = ref.route(zc, 1, normalize=False, active=active[a:b].cpu())
        assert torch.equal(ids, want) and ((r.weights[a:b].cpu().double() - w).abs() <= 2.0 ** -23 * w).all()
        want, mag = ref.route_gradient(dw[a:b].cpu(), zc, ids, "softmax", False, 1.0)
        assert ((dz[a:b].cpu().double() - want).abs() <= 64 * 2.0 ** -24 * mag + 2.0 ** -24 * want.abs() + 2.0 ** -150).all()


def test_experts_sums_of_more_features_than_a_launch_has_threads_for(mlxq):
    """2^34 results, four a thread."""
    T, K, N = 1048400, 32, 16388
    x, w = ref.random_mx(1, (T,), K, "e2m1", device="cuda"), ref.random_mx(2, (1, N), K, "e2m1", device="cuda")
    weights = torch.rand(T, 1, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    routing = mlxq.route_plan(torch.zeros(T, 1, dtype=torch.int32, device="cuda"), weights, 1)
    banner("mx_experts", T, K, N)
    y = mlxq.mx_experts(mlxq.Mx(*x), mlxq.Mx(*w), routing, combine=True)
    wv = ref.values(w)[0]
    border = 16777215 * 256 // 4097
    for rows in (slice(0, 20), slice(border - 10, border + 10), slice(T - 20, T)):
        xv, s = ref.values((x[0][rows], x[1][rows])), weights[rows].cpu().double()
        want = xv @ wv.t()
        tol = ref.product_bound(xv, wv, BF16, "e2m1")
        assert ((y[rows].cpu().double() - want * s).abs() <= tol * s + 2.0 ** -8 * (want.abs() + tol) * s * (1 + 2.0 ** -20) + 2.0 ** -133).all()
    del y
    torch.cuda.empty_cache()


class _Walled:
    """Memory for a result between two walls of 1 MB of a pattern, which must be there afterwards."""
    WALL = 1 << 20

    def __init__(self, nbytes):
        self.n = nbytes
        self.buf = torch.full((2 * self.WALL + -(-nbytes // 256) * 256,), 0xa5, dtype=torch.uint8, device="cuda")

    def ptr(self):
        return self.buf.data_ptr() + self.WALL

    def inside(self, dtype):
        return self.buf[self.WALL:self.WALL + self.n].view(dtype)

    def whole(self):
        return bool((self.buf[:self.WALL] == 0xa5).all()) and bool((self.buf[self.WALL + self.n:] == 0xa5).all())


# tiles of 16 and 32 rows, of 64, of 128 and of 256, whose results go by different ways
@pytest.mark.parametrize("T,k,E,K,N", [(40, 2, 4, 64, 33), (9, 3, 5, 416, 1100), (300, 2, 4, 160, 2050), (2100, 4, 3, 96, 1030), (6000, 2, 2, 64, 5001)])
@pytest.mark.parametrize("format", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_plan_writes_beside_the_results(mlxq, T, k, E, K, N, format, dtype):
    """starts and rows that are no plan's: results that mean nothing, and not a byte beside them or the workspace."""
    from mlxq import _lib
    lib, g = _lib.load(), torch.Generator().manual_seed(T)
    x = mlxq.mx_quantize(torch.randn(T, K, generator=g).cuda(), format)
    w = mlxq.mx_quantize(torch.randn(E, N, K, generator=g).cuda())
    ids = torch.randint(-1, E + 1, (T, k), generator=g, dtype=torch.int32).cuda()
    good = mlxq.route_plan(ids, torch.rand(T, k, generator=g).cuda(), E)
    M = T * k
    junk = torch.randint(-2 ** 31, 2 ** 31 - 1, (M,), generator=g, dtype=torch.int64).int().cuda()
    near = torch.randint(-3, M + 3, (M,), generator=g).int().cuda()
    st = lambda *v: torch.tensor([v[i % len(v)] for i in range(E + 1)], dtype=torch.int64).int().cuda()  # noqa: E731
    bad = [(st(-5, 10 ** 9, 3, -1, 2 ** 30), good.rows), (good.starts, torch.full_like(good.rows, 2 ** 30)), (good.starts, junk), (good.starts, near),
           (st(0, M, 0, M), near), (st(M - 1, 0), junk), (st(2 ** 31 - 1, -2 ** 31), near), (torch.zeros_like(good.starts), good.rows)]
    xv, _, keep_x = mlxq.mx._view("test", "x", x)
    wv, _, keep_w = mlxq.mx._view("test", "w", w)
    code = mlxq.mx._dt_of(dtype)
    for combine in (0, 1):
        need = lib.mlxq_mx_experts_workspace_size(T, k, N, combine, code)
        want = mlxq.mx_experts(x, w, good, combine=bool(combine), out_dtype=dtype)
        for i, (starts, rows) in enumerate(bad + [(good.starts, good.rows)]):
            banner("mx_experts", T, k, E, K, N, format, dtype, combine, i)
            y, ws = _Walled(want.numel() * want.element_size()), _Walled(need)
            routed = mlxq.mx._routed((ids, good.weights, starts, rows), T, k, E)
            _lib.check(lib.mlxq_mx_experts(ctypes.byref(xv), 0, K, ctypes.byref(wv), N, None, 0, ctypes.byref(routed), combine, y.ptr(), code,
                                           ws.ptr() if need else None, need, torch.cuda.current_stream().cuda_stream))
            assert y.whole() and ws.whole()
        assert torch.equal(y.inside(dtype).view(want.shape), want)  # the last one is a plan
    del keep_x, keep_w


def test_scales_padded_once(mlxq):
    """90 scales a row as a checkpoint stores them, and the same laid out once as Mx says: the one is copied by each call, the other
    goes to the library as it is."""
    import torch.nn.functional as F
    x = ref.random_mx(1, (3,), 2880, "e4m3", device="cuda")
    codes, scales = ref.random_mx(2, (4, 70), 2880, "e2m1", device="cuda")
    n = scales.shape[-1]
    assert n == 90
    held, rows = mlxq.Mx(codes, F.pad(scales, (0, -n % 4))[..., :n]), mlxq.Mx(x[0], F.pad(x[1], (0, -n % 4))[..., :n])
    routing = mlxq.route_plan(torch.tensor([[0, 3], [1, 2], [3, 0]], dtype=torch.int32, device="cuda"), torch.rand(3, 2, device="cuda"), 4)
    native = mlxq._lib.fast()
    code = mlxq.mx._dt_of(BF16)
    assert native.mx_experts(rows, mlxq.Mx(codes, scales), routing, None, False, code) is None
    y = native.mx_experts(rows, held, routing, None, False, code)
    assert y is not None and torch.equal(y, mlxq.mx_experts(mlxq.Mx(*x), mlxq.Mx(codes, scales), routing))
