"""mx_quantize, mx_dequantize, mx_matmul and mx_experts against their definitions (mx_ref), on the GPU."""
import itertools

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


def _wide(seed, rows, K, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g) * torch.exp(2 * torch.randn(rows, K // 32, 1, generator=g)).expand(-1, -1, 32).reshape(rows, K)
    return x.to(dtype)


def _edges(dtype):
    """Blocks whose maxima lie at the borders of two scales, ties of every code, zeros, subnormals, the largest and smallest
    values, infinities and NaN."""
    rows = []
    for top in (6.0, 6.25, 5.75, 448.0, 450.0, 447.0, 480.0, 1.0, 0.0, 2.0 ** -14, 2.0 ** -24):
        ties = [v * top / 448 for v in (0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 1.0625, 1.1875, 17.0, 19.0, 2 ** -10, 3 * 2 ** -10)]
        rows.append(([top, -top] + [s * v for v in ties for s in (1, -1)] + [-0.0, 0.0])[:32])
    big = torch.finfo(dtype).max
    for special in (float("inf"), float("-inf"), float("nan")):
        rows.append([special] + [1.0] * 31)
    rows.append([big, -big / 2] + [1.0] * 30)
    rows.append([torch.finfo(dtype).smallest_normal * 2 ** -3 * i for i in range(32)])
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    return x.reshape(4, -1)


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,K", [(1, 32), (1, 96), (3, 160), (5, 4096), (130, 2912), (2, 32 * 1027), (4, 0)])
def test_quantize_is_bit_exact(mlxq, format, dtype, rows, K):
    banner("mx_quantize", format, dtype, rows, K)
    x = _edges(dtype) if K == 0 else _wide(rows, rows, K, dtype)
    q = mlxq.mx_quantize(x.cuda(), format)
    code, scale = ref.quantized(x, format)
    assert torch.equal(ref.unpacked(q.codes), code)
    assert torch.equal(q.scales.cpu().long(), scale)
    if x.shape[1] % 128:  # up to a multiple of 4 the bytes between rows are 0
        pad = -(-x.shape[1] // 128) * 4 - x.shape[1] // 32
        whole = torch.as_strided(q.scales, (x.shape[0], x.shape[1] // 32 + pad), (x.shape[1] // 32 + pad, 1))
        assert not whole[:, x.shape[1] // 32:].any()


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
def test_quantize_strides(mlxq, format):
    """Slices, leading dimensions, broadcast rows, unaligned starts, a column slice: as a contiguous copy."""
    base = _wide(1, 24, 512, BF16).cuda()
    for x in (base[:, 64:192], base[::3], base.view(2, 12, 512)[:, 3:7, 32:96], base[:1].expand(5, 512), base[:, 4:68], base[4],
              base.view(2, 3, 4, 512).transpose(0, 2)):
        a, b = mlxq.mx_quantize(x, format), mlxq.mx_quantize(x.contiguous().clone(), format)
        assert a.codes.shape[:-1] == x.shape[:-1] and torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8))
        assert torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_dequantize(mlxq, format, dtype):
    """Every code under every scale, rounded once."""
    n = 16 if format == "e2m1" else 256
    code = torch.arange(n).repeat(256, 32 * 16 // n if n <= 512 else 1)[:, :512]
    scales = torch.arange(256)[:, None].expand(-1, 16).to(torch.uint8).contiguous()
    mx = mlxq.Mx(ref.packed(code, format).cuda(), scales.cuda())
    got, want = mlxq.mx_dequantize(mx, dtype).cpu(), ref.values((mx.codes, mx.scales)).to(dtype)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])


def test_empty(mlxq):
    for format in ("e2m1", "e4m3"):
        q = mlxq.mx_quantize(torch.empty(0, 64, device="cuda"), format)
        assert q.codes.shape[0] == 0 and mlxq.mx_dequantize(q).shape == (0, 64)
        w = mlxq.mx_quantize(torch.randn(5, 64, device="cuda"))
        assert mlxq.mx_matmul(q, w).shape == (0, 5)
        assert mlxq.mx_matmul(mlxq.mx_quantize(torch.randn(3, 64, device="cuda"), format), mlxq.Mx(w.codes[:0], w.scales[:0])).shape == (3, 0)


SHAPES = [(1, 32, 1), (1, 4096, 16), (2, 96, 17), (7, 160, 33), (15, 2912, 70), (16, 128, 640), (17, 416, 130), (33, 1024, 48),
          (63, 288, 100), (64, 544, 260), (65, 96, 65), (100, 1312, 300), (129, 128, 520), (257, 672, 130), (300, 224, 3000), (1030, 160, 2100),
          # more features than 256 workgroups of the smallest tiles have: every other tile
          (5, 160, 6001), (16, 96, 12010), (11, 288, 20003), (20, 160, 5000), (32, 96, 20010), (100, 160, 12001), (150, 288, 14002), (200, 160, 20001),
          (3001, 160, 9003), (2100, 800, 12301),
          # groups of waves that split K, with runs of several steps and some without
          (60, 2912, 1900), (250, 1312, 1000), (100, 2912, 4000), (250, 2912, 3900), (500, 1312, 4000)]


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_matmul(mlxq, format, M, K, N):
    """Every result within what its sums and its rounding may be off by, in the three types, with and without a bias."""
    x, w = ref.random_mx(M + K, (M,), K, format), ref.random_mx(N, (N,), K, "e2m1")
    xv, wv = ref.values(x), ref.values(w)
    want = xv @ wv.t()
    xd, wd = mlxq.Mx(x[0].cuda(), x[1].cuda()), mlxq.Mx(w[0].cuda(), w[1].cuda())
    bias = torch.randn(N, generator=torch.Generator().manual_seed(3)) * want.abs().mean().item()
    for dtype, b in itertools.product((F32, BF16, F16), (None, bias, bias.to(BF16))):
        banner("mx_matmul", format, M, K, N, dtype, None if b is None else b.dtype)
        y = mlxq.mx_matmul(xd, wd, None if b is None else b.cuda(), dtype)
        assert y.dtype == dtype and y.shape == (M, N)
        exact = want if b is None else want + b.double()
        tol = ref.product_bound(xv, wv, dtype, format) + (0 if b is None else (UNIT_SUM + ref.UNIT[dtype]) * (b.double().abs() + want.abs()))
        fits = exact.abs() < torch.finfo(dtype).max
        assert ((y.cpu().double() - exact).abs() <= tol)[fits].all()
        if dtype != F32 and b is not None:
            break


UNIT_SUM = 2.0 ** -23  # the addition of the bias in f32


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
def test_matmul_large_result(mlxq, format):
    """A result past 2^31 values, whose rows end inside a piece of eight: rows at the start, at the border and at the end."""
    M, K, N = 66001, 64, 32771
    x, w = ref.random_mx(1, (M,), K, format), ref.random_mx(2, (N,), K, "e2m1")
    banner("mx_matmul", format, M, K, N)
    y = mlxq.mx_matmul(mlxq.Mx(x[0].cuda(), x[1].cuda()), mlxq.Mx(w[0].cuda(), w[1].cuda()), out_dtype=BF16)
    border = 2 ** 31 // N
    for rows in (slice(0, 20), slice(border - 10, border + 10), slice(M - 20, M)):
        xv, wv = ref.values((x[0][rows], x[1][rows])), ref.values(w)
        assert ((y[rows].cpu().double() - xv @ wv.t()).abs() <= ref.product_bound(xv, wv, BF16, format)).all()


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("M", [3, 40, 200])
def test_matmul_special_scales(mlxq, format, M):
    """NaN blocks make their rows and columns NaN and nothing else; the smallest and large scales are as exact as others."""
    K, N = 288, 96
    x, w = ref.random_mx(1, (M,), K, format), ref.random_mx(2, (N,), K, "e2m1")
    x[1][0, 4], x[1][1], x[1][2] = 255, 0, 230
    w[1][5, 8], w[1][6], w[1][7] = 255, 0, 227
    xv, wv = ref.values(x), ref.values(w)
    want = xv @ wv.t()
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[0], nan[:, 5] = True, True
    # sums whose terms pass f32's range (row 2 by column 7) overflow on the way: an infinity, or the difference of two
    over = torch.nan_to_num(xv).abs() @ torch.nan_to_num(wv).abs().t() > torch.finfo(F32).max / 2
    for dtype in (F32, BF16):
        y = mlxq.mx_matmul(mlxq.Mx(x[0].cuda(), x[1].cuda()), mlxq.Mx(w[0].cuda(), w[1].cuda()), out_dtype=dtype).cpu()
        assert not (y.isnan() & ~nan & ~over).any() and y[nan].isnan().all()
        fits = ~nan & ~over & (want.abs() < torch.finfo(dtype).max / 2)
        tol = ref.product_bound(torch.nan_to_num(xv), torch.nan_to_num(wv), dtype, format)
        assert ((y.double() - want).abs() <= tol + 2.0 ** -126)[fits].all()


def test_scales_between_rows_hold_anything(mlxq):
    """The bytes between rows' scales are not read for a result: NaN there changes nothing."""
    for M, format in ((1, "e4m3"), (5, "e4m3"), (40, "e2m1"), (300, "e4m3"), (300, "e2m1")):
        K, N = 416, 200  # 13 scales a row
        x, w = ref.random_mx(1, (M,), K, format, device="cuda"), ref.random_mx(2, (N,), K, "e2m1", device="cuda")
        got = []
        for fill in (0, 255):
            pads = []
            for codes, scales in (x, w):
                room = torch.full((scales.shape[0], 20), fill, dtype=torch.uint8, device="cuda")
                room[:, :13] = scales
                pads.append(mlxq.Mx(codes, room[:, :13]))
            got.append(mlxq.mx_matmul(*pads, out_dtype=F32))
        # contiguous scales, whose rows start at odd addresses, are copied
        got.append(mlxq.mx_matmul(mlxq.Mx(*x), mlxq.Mx(*w), out_dtype=F32))
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]) and not got[0].isnan().any()


def test_leading_dimensions_and_fast_path(mlxq, monkeypatch):
    """Both call paths give the same, over leading dimensions."""
    from mlxq import _lib
    x = mlxq.mx_quantize(torch.randn(2, 3, 5, 160, device="cuda"), "e4m3")
    w, b = mlxq.mx_quantize(torch.randn(40, 160, device="cuda")), torch.randn(40, device="cuda")
    fast = mlxq.mx_matmul(x, w, b), mlxq.mx_dequantize(x), mlxq.mx_quantize(torch.ones(3, 64, device="cuda")).scales
    monkeypatch.setattr(_lib, "_fast", _lib._NoFast())
    slow = mlxq.mx_matmul(x, w, b), mlxq.mx_dequantize(x), mlxq.mx_quantize(torch.ones(3, 64, device="cuda")).scales
    assert all(torch.equal(a, c) for a, c in zip(fast, slow)) and fast[0].shape == (2, 3, 5, 40)


def _ids(seed, T, k, E, lost=0.2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int()
    out = torch.rand(T, k, generator=g) < lost
    return torch.where(out, torch.where(torch.rand(T, k, generator=g) < 0.5, -1, E + 3).int(), ids)


EXPERTS = [(1, 1, 1, 32, 5, False), (1, 4, 32, 160, 40, False), (3, 4, 8, 288, 70, True), (17, 2, 5, 96, 33, False), (70, 3, 4, 416, 130, True),
           (90, 2, 3, 1056, 48, False), (200, 4, 4, 224, 300, True), (400, 2, 3, 160, 520, False), (33, 8, 60, 128, 24, False)]


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("T,k,E,K,N,per", EXPERTS)
@pytest.mark.parametrize("lost", [0.0, 0.3, 1.0])
def test_experts(mlxq, format, T, k, E, K, N, per, lost):
    """Each choice's product, zeros without an expert, and the weighted sums; experts with no row, one and many."""
    x, w = ref.random_mx(T, (T, k) if per else (T,), K, format, 122, 129), ref.random_mx(E, (E, N), K, "e2m1", 122, 129)
    ids = _ids(T, T, k, E, lost)
    g = torch.Generator().manual_seed(1)
    weights = torch.rand(T, k, generator=g)
    bias = torch.randn(E, N, generator=g)
    want, xv, wv = ref.experts(x, w, ids, bias)
    rows = xv if per else xv[:, None].expand(-1, k, -1)
    routing = mlxq.route_plan(ids.cuda(), weights.cuda(), E)
    xd, wd = mlxq.Mx(x[0].cuda(), x[1].cuda()), mlxq.Mx(w[0].cuda(), w[1].cuda())
    live = (ids >= 0) & (ids < E)
    for dtype in (F32, BF16, F16):
        banner("mx_experts", format, T, k, E, K, N, per, lost, dtype)
        tol = torch.zeros_like(want)
        for t in range(T):
            for j in range(k):
                if live[t, j]:
                    tol[t, j] = ref.product_bound(rows[t, j:j + 1], wv[ids[t, j]], dtype, format)[0]
        tol += live[..., None] * (UNIT_SUM + ref.UNIT[dtype]) * (want.abs() + 2 * bias.abs().max())
        y = mlxq.mx_experts(xd, wd, routing, bias.cuda(), out_dtype=dtype).cpu().double()
        assert y.shape == (T, k, N) and ((y - want).abs() <= tol).all()
        total = mlxq.mx_experts(xd, wd, routing, bias.cuda(), combine=True, out_dtype=dtype).cpu().double()
        exact = (want * weights.double()[..., None]).sum(1)
        # k products of f32 weights and rounded results, summed in f32, rounded once
        mag = ((want.abs() + tol) * weights.double()[..., None]).sum(1)
        bound = (tol * weights.double()[..., None]).sum(1) + (k + 1) * 2.0 ** -23 * mag + ref.UNIT[dtype] * mag + ref.TINY[dtype]
        assert total.shape == (T, N) and ((total - exact).abs() <= bound).all()
        if T > 100:
            break


def test_experts_skewed(mlxq):
    """All tokens at one expert, and one token at each of many."""
    E, K, N = 16, 160, 96
    x, w = ref.random_mx(1, (300,), K, "e4m3", 122, 129), ref.random_mx(2, (E, N), K, "e2m1", 122, 129)
    xv, wv = ref.values(x), ref.values(w)
    xd, wd = mlxq.Mx(x[0].cuda(), x[1].cuda()), mlxq.Mx(w[0].cuda(), w[1].cuda())
    for ids in (torch.full((300, 1), 11, dtype=torch.int32), (torch.arange(300, dtype=torch.int32) % E)[:, None]):
        routing = mlxq.route_plan(ids.cuda(), torch.ones(300, 1).cuda(), E)
        y = mlxq.mx_experts(xd, wd, routing, out_dtype=F32).cpu().double()[:, 0]
        want = torch.bmm(wv[ids[:, 0].long()], xv[:, :, None])[..., 0]
        for t in range(300):
            assert ((y[t] - want[t]).abs() <= ref.product_bound(xv[t:t + 1], wv[int(ids[t])], F32, "e4m3")[0]).all()


def test_a_broken_plan_stays_in_bounds(mlxq):
    """starts and rows that are no plan: wrong results, but nothing is read or written outside the operands."""
    T, k, E, K, N = 40, 2, 4, 64, 32
    x = mlxq.mx_quantize(torch.randn(T, K, device="cuda"), "e4m3")
    w = mlxq.mx_quantize(torch.randn(E, N, K, device="cuda"))
    good = mlxq.route_plan(_ids(1, T, k, E, 0).cuda(), torch.rand(T, k).cuda(), E)
    guard = torch.full((3, T, k, N), 7.0, device="cuda", dtype=BF16)
    for starts, rows in ((torch.tensor([-5, 10 ** 9, 3, -1, 2 ** 30]), good.rows), (good.starts, torch.full_like(good.rows, 2 ** 30)),
                         (good.starts, torch.full_like(good.rows, -7)), (torch.tensor([70, 60, 50, 40, 30]), good.rows)):
        bad = mlxq.Routing(good.ids, good.weights, starts.int().cuda(), rows.int())
        mlxq.mx_experts(x, w, bad)
        mlxq.mx_experts(x, w, bad, combine=True)
    torch.cuda.synchronize()
    assert (guard == 7).all()
    assert torch.equal(mlxq.mx_experts(x, w, good), mlxq.mx_experts(x, w, mlxq.route_plan(good.ids, good.weights, E)))


def test_overlapping_runs_of_many_choices(mlxq):
    """Starts of 512 runs that each hold all of 2^25 choices: more tiles than 2^31.  Results mean nothing; memory is left alone."""
    T, k, E = 2 ** 19, 64, 1024
    x = mlxq.Mx(torch.zeros(T, 16, dtype=torch.uint8, device="cuda"), torch.full((T, 4), 127, dtype=torch.uint8, device="cuda")[:, :1])
    w = mlxq.Mx(torch.zeros(E, 1, 16, dtype=torch.uint8, device="cuda"), torch.full((E, 1, 4), 127, dtype=torch.uint8, device="cuda")[..., :1])
    starts = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    starts[1::2] = T * k
    routing = mlxq.Routing(torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda"), starts,
                           torch.arange(T * k, dtype=torch.int32, device="cuda"))
    y = mlxq.mx_experts(x, w, routing)
    assert not y[:1000].any()
    # and a plan after it is as good as ever
    good = mlxq.route_plan(routing.ids[:100], routing.weights[:100], E)
    assert torch.equal(good.rows.cpu(), torch.arange(6400, dtype=torch.int32))


def test_repeated_calls_and_streams(mlxq):
    """The same bits on any stream and from call to call, with other calls between."""
    x = mlxq.mx_quantize(torch.randn(500, 1056, device="cuda"), "e4m3")
    w = mlxq.mx_quantize(torch.randn(900, 1056, device="cuda"))
    first = mlxq.mx_matmul(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = [mlxq.mx_matmul(x, w) for _ in range(3)]
    mine = [mlxq.mx_matmul(x, w) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, t) for t in other + mine)


def test_past_32_bits(mlxq):
    """Operands and results past 4 GiB: sampled rows at both ends."""
    g = torch.Generator(device="cuda").manual_seed(0)
    # 4.5 GB of bf16 through quantisation and back
    x = torch.randn(36000, 65536, generator=g, device="cuda", dtype=BF16)
    q = mlxq.mx_quantize(x, "e4m3")
    for r in (0, 17999, 35999):
        code, scale = ref.quantized(x[r:r + 1].cpu(), "e4m3")
        assert torch.equal(ref.unpacked(q.codes[r:r + 1]), code) and torch.equal(q.scales[r:r + 1].cpu().long(), scale)
    back = mlxq.mx_dequantize(q)
    assert torch.equal(back[35999].cpu().double(), ref.values((q.codes[35999:], q.scales[35999:]))[0])
    del x, back
    # 2.4 GB of e4m3 rows, 4.6 GB of results
    m = mlxq.Mx(q.codes, q.scales)
    w = ref.random_mx(5, (64000,), 65536 // 512, "e2m1", device="cuda")  # K = 128
    cut = mlxq.mx_quantize(torch.randn(36000, 128, generator=g, device="cuda"), "e4m3")
    y = mlxq.mx_matmul(cut, mlxq.Mx(*w))
    wv = ref.values(w)
    for r in (0, 33554, 35999):
        xv = ref.values((cut.codes[r:r + 1], cut.scales[r:r + 1]))
        assert ((y[r].cpu().double() - (xv @ wv.t())[0]).abs() <= ref.product_bound(xv, wv, BF16, "e4m3")[0]).all()
    del y
    few = mlxq.mx_quantize(torch.randn(20, 65536, generator=g, device="cuda"))
    y = mlxq.mx_matmul(m, few, out_dtype=F32)
    fv = ref.values(few)
    for r in (0, 35999):
        xv = ref.values((m.codes[r:r + 1], m.scales[r:r + 1]))
        assert ((y[r].cpu().double() - (xv @ fv.t())[0]).abs() <= ref.product_bound(xv, fv, F32, "e4m3")[0]).all()
