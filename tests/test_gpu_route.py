"""route_experts, route_plan and route_experts_backward against their definitions (mx_ref), on the GPU."""
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


def _logits(seed, T, E, dtype, std=1.5):
    return (torch.randn(T, E, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _check(mlxq, z, k, **kw):
    bias, active = kw.get("bias"), kw.get("active")
    got = mlxq.route_experts(z.cuda(), k, kw.get("scoring", "softmax"), bias=None if bias is None else bias.cuda(),
                             groups=kw.get("groups", 1), kept_groups=kw.get("kept", 1), group_best=kw.get("best", 1),
                             normalize=kw.get("normalize", True), scale=kw.get("scale", 1.0), active=None if active is None else active.cuda())
    ids, w = ref.route(z, k, **kw)
    starts, rows = ref.plan(ids, z.shape[1])
    assert torch.equal(got.ids.cpu(), ids)
    # taken in 64 bits, rounded once, but that sums of 1024 scores may be off by 2^-42
    g = got.weights.cpu().double()
    assert torch.equal(g.isnan(), w.isnan()) and ((g - w).abs() <= (2.0 ** -24 + 2.0 ** -40) * w.abs() + 2.0 ** -149)[~w.isnan()].all()
    assert torch.equal(got.starts.cpu(), starts) and torch.equal(got.rows.cpu(), rows)
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 5, 5), (17, 60, 4), (5, 64, 8), (66, 65, 6), (9, 128, 64), (40, 160, 6), (7, 256, 8),
                                   (4, 384, 10), (3, 513, 3), (2, 1024, 33)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_routing(mlxq, dtype, T, E, k, scoring):
    banner("route_experts", dtype, T, E, k, scoring)
    z = _logits(T + E, T, E, dtype)
    bias = 0.2 * torch.randn(E, generator=torch.Generator().manual_seed(2))
    active = torch.rand(T, generator=torch.Generator().manual_seed(3)) > 0.3
    _check(mlxq, z, k, scoring=scoring)
    _check(mlxq, z, k, scoring=scoring, normalize=False, scale=2.5)
    _check(mlxq, z, k, scoring=scoring, bias=bias, active=active)
    for groups in (2, 4, 8):
        if E % groups == 0:
            for kept in {1, groups // 2, groups}:
                if k <= kept * (E // groups):
                    for best in (1, 2):
                        _check(mlxq, z, k, scoring=scoring, groups=groups, kept=kept, best=best)
                        _check(mlxq, z, k, scoring=scoring, groups=groups, kept=kept, best=best, bias=bias, normalize=False)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_ties_go_to_the_lowest_expert(mlxq, scoring):
    """Few different logits, zeros of both signs, saturated scores, and biases that are equal too."""
    g = torch.Generator().manual_seed(1)
    z = torch.randint(-2, 3, (60, 96), generator=g).float()
    z[::2] = torch.where(z[::2] == 0, -0.0, z[::2])
    bias = torch.randint(0, 2, (96,), generator=g).float()
    for k in (1, 7):
        _check(mlxq, z, k, scoring=scoring)
        _check(mlxq, z, k, scoring=scoring, bias=bias)
        _check(mlxq, z, k, scoring=scoring, groups=8, kept=3, best=2)
        _check(mlxq, z, k, scoring=scoring, groups=8, kept=3, best=1, bias=bias)
    if scoring == "sigmoid":  # scores of 1 in 64 bits: without a bias the logits still decide
        _check(mlxq, z * 40, 5, scoring=scoring)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_and_undefined_logits(mlxq, scoring):
    z = _logits(4, 12, 48, F32)
    z[0, :40] = float("-inf")
    z[1] = float("-inf")
    z[2, 3:] = float("-inf")
    z[3] = torch.finfo(F32).min
    z[4, 7] = float("nan")
    z[5, 9] = float("inf")
    z[6, 4:] = float("nan")
    z[7] = float("nan")
    z[8] = torch.finfo(F32).max
    for k in (2, 6):
        for kw in ({}, {"normalize": False}, {"groups": 4, "kept": 2}):
            _check(mlxq, z, k, scoring=scoring, **kw)
    active = torch.ones(12, dtype=torch.bool)
    active[[1, 4, 7]] = False
    got = _check(mlxq, z, 3, scoring=scoring, active=active)
    assert (got.ids[7].cpu() == -1).all() and (got.weights[7].cpu() == 0).all()


def test_strides_and_paths(mlxq, monkeypatch):
    from mlxq import _lib
    z = _logits(5, 30, 80, BF16).cuda()
    for x in (z[:, :64], z[::3], z.t()[:20].t(), z[:1].expand(7, 80), z[:, 5:69]):
        a, b = mlxq.route_experts(x, 4), mlxq.route_experts(x.contiguous(), 4)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    bias = torch.randn(80).cuda()
    fast = mlxq.route_experts(z, 4, "sigmoid", bias=bias, groups=4, kept_groups=2, group_best=2, scale=2)
    dw = torch.randn(30, 4, device="cuda")
    grad = mlxq.route_experts_backward(dw, z, fast.ids, "sigmoid", scale=2)
    monkeypatch.setattr(_lib, "_fast", _lib._NoFast())
    slow = mlxq.route_experts(z, 4, "sigmoid", bias=bias, groups=4, kept_groups=2, group_best=2, scale=2)
    assert all(torch.equal(p, q) for p, q in zip(fast, slow))
    assert torch.equal(grad, mlxq.route_experts_backward(dw, z, fast.ids, "sigmoid", scale=2))


@pytest.mark.parametrize("n,k,E", [(1, 1, 1), (5, 3, 7), (63, 1, 64), (64, 1, 2), (65, 2, 9), (1023, 2, 33), (1024, 2, 3), (700, 3, 1024), (4099, 8, 60),
                                   (9000, 8, 128), (70001, 2, 256), (40000, 8, 5), (30001, 5, 1024),
                                   (300007, 1, 100)])
@pytest.mark.parametrize("lost", [0.0, 0.25, 1.0])
def test_plan(mlxq, n, k, E, lost):
    banner("route_plan", n, k, E, lost)
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, E, (n, k), generator=g, dtype=torch.int32)
    out = torch.rand(n, k, generator=g) < lost
    ids = torch.where(out, torch.randint(0, 2, (n, k), generator=g, dtype=torch.int32) * (E + 1) - 1, ids)  # -1 or E
    r = mlxq.route_plan(ids.cuda(), torch.rand(n, k).cuda(), E)
    key = torch.where((ids >= 0) & (ids < E), ids, E).flatten()
    assert torch.equal(r.rows.cpu().long(), torch.sort(key, stable=True).indices)
    want = torch.tensor([int((key < e).sum()) for e in range(E + 1)], dtype=torch.int32)
    assert torch.equal(r.starts.cpu(), want)


def test_many_tokens(mlxq):
    """Enough for many workgroups, against the definition at sampled tokens and the plan by sorting."""
    z = _logits(6, 40000, 128, BF16)
    active = torch.rand(40000, generator=torch.Generator().manual_seed(1)) > 0.1
    r = mlxq.route_experts(z.cuda(), 8, active=active.cuda())
    at = torch.arange(0, 40000, 997)
    ids, w = ref.route(z[at], 8, active=active[at])
    assert torch.equal(r.ids.cpu()[at], ids) and ((r.weights.cpu()[at].double() - w).abs() <= 2.0 ** -23 * w).all()
    key = torch.where(r.ids >= 0, r.ids, 128).flatten()
    assert torch.equal(r.rows.long(), torch.sort(key, stable=True).indices)
    assert torch.equal(r.starts.long(), torch.searchsorted(torch.sort(key).values, torch.arange(129, device="cuda", dtype=torch.int32)))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (3, 8, 2), (20, 60, 6), (9, 64, 64), (33, 130, 8), (5, 256, 8), (4, 500, 3), (3, 1024, 12)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
def test_gradient(mlxq, dtype, T, E, k, scoring, normalize):
    banner("route_experts_backward", dtype, T, E, k, scoring, normalize)
    z = _logits(T, T, E, dtype)
    g = torch.Generator().manual_seed(2)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int()
    ids = torch.where(torch.rand(T, k, generator=g) < 0.15, torch.where(torch.rand(T, k, generator=g) < 0.5, -1, E).int(), ids)
    dw = torch.randn(T, k, generator=g)
    got = mlxq.route_experts_backward(dw.cuda(), z.cuda(), ids.cuda(), scoring, normalize, 1.7)
    want, mag = ref.route_gradient(dw, z, ids, scoring, normalize, 1.7)
    # scores: the exponential's 4 roundings, a sum of 16 a lane and 6 steps, a division; each of the three sums over the
    # choices 6 steps; some ten products: below 64 roundings of the terms
    assert got.dtype == dtype and ((got.cpu().double() - want).abs() <= 64 * 2.0 ** -24 * mag + ref.UNIT[dtype] * want.abs() + ref.TINY[dtype]).all()


def test_gradient_is_that_of_differences(mlxq):
    """Central differences of the definition in 64 bits, the choice held: h^2 / 6 of a third derivative below 8 times the
    gradient's terms, and rounding of 2^-50 over h."""
    h = 2.0 ** -11
    for scoring, normalize in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        z, dw = _logits(1, 2, 12, F32), torch.randn(2, 3, generator=torch.Generator().manual_seed(2))
        ids, _ = ref.route(z, 3)
        got = mlxq.route_experts_backward(dw.cuda(), z.cuda(), ids.cuda(), scoring, normalize, 2.0).cpu().double()
        _, mag = ref.route_gradient(dw, z, ids, scoring, normalize, 2.0)

        def f(z):
            s = torch.sigmoid(z) if scoring == "sigmoid" else torch.softmax(z, -1)
            p = s.gather(1, ids.long())
            return float((2.0 * (p / p.sum(-1, keepdim=True) if normalize else p) * dw.double()).sum())
        for t in range(2):
            for e in range(12):
                up, dn = z.double().clone(), z.double().clone()
                up[t, e] += h
                dn[t, e] -= h
                slack = h * h / 6 * 8 * float(dw.abs().sum()) * 2 + 2.0 ** -50 * 20 / h
                assert abs(float(got[t, e]) - (f(up) - f(dn)) / (2 * h)) <= 64 * 2.0 ** -24 * float(mag[t, e]) + slack


def test_gradient_of_masked_logits(mlxq):
    """-infinity has a score and a gradient of 0."""
    z = _logits(3, 4, 40, F32)
    z[0, 10:] = float("-inf")
    z[1] = float("-inf")
    for scoring in ("softmax", "sigmoid"):
        for normalize in (True, False):
            ids, _ = ref.route(z, 4, scoring)
            dw = torch.randn(4, 4, generator=torch.Generator().manual_seed(1))
            got = mlxq.route_experts_backward(dw.cuda(), z.cuda(), ids.cuda(), scoring, normalize).cpu()
            assert got.isfinite().all() and not got[0, 10:].any() and not got[1].any()


def test_empty(mlxq):
    r = mlxq.route_experts(torch.empty(0, 16, device="cuda"), 2)
    assert r.ids.shape == (0, 2) and r.starts.tolist() == [0] * 17 and r.rows.numel() == 0
    assert mlxq.route_experts_backward(torch.empty(0, 2, device="cuda"), torch.empty(0, 16, device="cuda"), r.ids).shape == (0, 16)
    x = mlxq.mx_quantize(torch.empty(0, 64, device="cuda"), "e4m3")
    w = mlxq.mx_quantize(torch.randn(16, 8, 64, device="cuda"))
    assert mlxq.mx_experts(x, w, r).shape == (0, 2, 8) and mlxq.mx_experts(x, w, r, combine=True).shape == (0, 8)
