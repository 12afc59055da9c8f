"""Routing where scores leave f32's range, and tokens that go nowhere: against definitions of its own, in 64 bits."""
import pytest
import torch
import torch.nn.functional as F

import mx_ref as ref
from gpu_util import banner

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mlxq():
    import mlxq as m
    m.load()
    return m


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def _normalized_weights(z, ids, scoring, scale):
    """w = scale s / (sum of s over the chosen) from the logarithms of the scores, which stay in range."""
    s = F.logsigmoid(z.double()) if scoring == "sigmoid" else z.double()
    return scale * torch.softmax(s.gather(1, ids.long()), -1)


def _normalized_gradient(dw, z, ids, scoring, scale):
    """(dz, a bound of what its terms come to): dz_j = w_j (dw_j - sum dw w / scale) times 1 - s_j of a sigmoid."""
    share, d = _normalized_weights(z, ids, scoring, 1.0), dw.double() * scale
    q = torch.sigmoid(-z.double().gather(1, ids.long())) if scoring == "sigmoid" else 1.0
    put = lambda v: torch.zeros(z.shape, dtype=torch.float64).scatter_(1, ids.long(), v)  # noqa: E731
    return put(share * (d - (share * d).sum(-1, keepdim=True)) * q), put(share * (d.abs() + (share * d.abs()).sum(-1, keepdim=True)) * q)


def _far_rows(scoring, E, k, dtype):
    """Rows whose chosen experts all lie far below 0 (sigmoid), or below the row's largest logit (softmax), by 0 to 700, some
    close together and some 40 apart."""
    far = [0, 30, 80, 86, 87, 88, 90, 95, 100, 104, 130, 200, 300, 500, 700]
    if dtype == F16:
        far = [v for v in far if v <= 500]
    T = 2 * len(far)
    z = _randn(E, T, E)
    ids = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).int()
    for t in range(T):
        spread = torch.linspace(0, 40, k) if t % 2 else _randn(t, k)
        z[t, ids[t].long()] = -float(far[t // 2]) - spread + (20.0 if scoring == "softmax" else 0.0)
        if scoring == "softmax":
            others = [e for e in range(E) if e not in ids[t].tolist()]
            z[t, others[0]] = 20.0 + (0.0 if t % 4 else 2.0)
    return z.to(dtype), ids


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("E,k", [(8, 2), (60, 6), (256, 8), (1024, 3)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_gradient_of_choices_far_below(mlxq, dtype, E, k, scoring):
    """Normalized weights are ordinary numbers however small the scores are, and so is their gradient."""
    banner("route_experts_backward", dtype, E, k, scoring)
    z, ids = _far_rows(scoring, E, k, dtype)
    dw = 3 * _randn(5, *ids.shape)
    got = mlxq.route_experts_backward(dw.cuda(), z.cuda(), ids.cuda(), scoring, True, 1.7)
    want, mag = _normalized_gradient(dw, z, ids, scoring, 1.7)
    # 64 roundings as for ordinary scores (test_gpu_route.py); a difference of logits of up to 40 + 8 is rounded before its exponential
    tol = (64 + 48) * 2.0 ** -24 * mag + ref.UNIT[dtype] * want.abs() + ref.TINY[dtype]
    assert got.dtype == dtype and ((got.cpu().double() - want).abs() <= tol).all()


def test_gradient_of_choices_far_below_is_that_of_differences(mlxq):
    """Central differences of the weights in 64 bits: h^2 / 6 of a third derivative below 8 times the gradient's terms."""
    h = 2.0 ** -11
    for scoring in ("softmax", "sigmoid"):
        z, ids = _far_rows(scoring, 12, 3, F32)
        dw = _randn(2, *ids.shape)
        got = mlxq.route_experts_backward(dw.cuda(), z.cuda(), ids.cuda(), scoring, True, 2.0).cpu().double()
        _, mag = _normalized_gradient(dw, z, ids, scoring, 2.0)
        f = lambda v: (_normalized_weights(v, ids, scoring, 2.0) * dw.double()).sum(-1)  # noqa: E731
        for e in range(12):
            up, dn = z.double().clone(), z.double().clone()
            up[:, e] += h
            dn[:, e] -= h
            slack = h * h / 6 * 8 * 2 * dw.double().abs().sum(-1) + 2.0 ** -50 * 1000 / h
            assert ((got[:, e] - (f(up) - f(dn)) / (2 * h)).abs() <= 112 * 2.0 ** -24 * mag[:, e] + slack).all()


def test_gradient_follows_the_router(mlxq):
    """A bias takes tokens to experts far below their largest logit: the gradient of the weights that route_experts gives."""
    E, k = 40, 4
    z = _randn(1, 50, E)
    z[:, :10] += 120
    bias = torch.cat([torch.zeros(20), torch.full((20,), 5.0)])
    r = mlxq.route_experts(z.cuda(), k, "softmax", bias=bias.cuda())
    ids = r.ids.cpu()
    assert (ids >= 20).all()
    want = _normalized_weights(z, ids, "softmax", 1.0)
    assert ((r.weights.cpu().double() - want).abs() <= 2.0 ** -23 * want).all()
    dw = _randn(3, 50, k)
    got = mlxq.route_experts_backward(dw.cuda(), z.cuda(), r.ids).cpu().double()
    want, mag = _normalized_gradient(dw, z, ids, "softmax", 1.0)
    assert ((got - want).abs() <= (72 * 2.0 ** -24) * mag + 2.0 ** -24 * want.abs() + 2.0 ** -150).all()


def test_no_weight_has_no_gradient(mlxq):
    """Where the chosen scores are 0 in 64 bits the weights are 0, and so is their gradient."""
    z = _randn(1, 4, 16)
    z[0, :4], z[1, :4], z[2, :4], z[3, :4] = -800.0, torch.finfo(F32).min, float("-inf"), -746.0
    ids = torch.arange(4, dtype=torch.int32).repeat(4, 1)
    for scoring in ("softmax", "sigmoid"):
        bias = torch.full((16,), -1.0)
        bias[:4] = 4.0
        r = mlxq.route_experts(z.cuda(), 4, scoring, bias=bias.cuda())
        assert (r.ids.sort(-1).values.cpu() == ids).all() and not r.weights.any()
        assert not mlxq.route_experts_backward(torch.randn(4, 4).cuda(), z.cuda(), ids.cuda(), scoring).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
def test_tokens_without_an_expert_pass_nothing_on(mlxq, dtype, scoring, normalize):
    """Rows of a padded batch may hold anything; so may the logits of experts that a sigmoid's token did not choose."""
    z = _randn(1, 8, 96).to(dtype)
    z[1], z[2, 5], z[3], z[4, 70] = float("nan"), float("nan"), float("inf"), float("inf")
    active = torch.tensor([True, False, False, False, False, True, True, True])
    r = mlxq.route_experts(z.cuda(), 4, scoring, normalize=normalize, active=active.cuda())
    dw = _randn(2, 8, 4)
    dw[1] = float("nan")
    got = mlxq.route_experts_backward(dw.cuda(), z.cuda(), r.ids, scoring, normalize).cpu()
    assert not got[~active].any() and got.isfinite().all() and got[active].any(-1).all()
    alone = mlxq.route_experts_backward(dw[active].cuda(), z[active].cuda(), r.ids[active.cuda()], scoring, normalize).cpu()
    assert torch.equal(got[active], alone)
    if scoring == "sigmoid":
        ids = torch.tensor([[3, 9, 40, 95]], dtype=torch.int32)
        y = z[5:6].clone()
        y[0, 7], y[0, 50] = float("nan"), float("inf")
        clean = mlxq.route_experts_backward(dw[5:6].cuda(), z[5:6].cuda(), ids.cuda(), scoring, normalize)
        assert torch.equal(mlxq.route_experts_backward(dw[5:6].cuda(), y.cuda(), ids.cuda(), scoring, normalize), clean)


def _undefined_choice(zt, k, groups, kept):
    """The choice of a softmax's row that holds a NaN or +infinity: by its logits alone, NaN last, a group by its best."""
    E = len(zt)
    size = E // groups
    low = [v if v == v else float("-inf") for v in zt]
    best = [max(low[g * size:(g + 1) * size]) for g in range(groups)]
    keep = sorted(range(groups), key=lambda g: (-best[g], g))[:kept] if kept < groups else range(groups)
    allowed = [e for e in range(E) if e // size in keep]
    return sorted(allowed, key=lambda e: (zt[e] != zt[e], -low[e], e))[:k]


@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_choice_of_undefined_rows(mlxq, scoring, biased, best):
    """NaN logits come after all others, with a bias and in groups too; other rows are as ever."""
    E = 48
    z = _randn(4, 14, E)
    z[1, 7] = float("nan")
    z[2, 9] = float("inf")
    z[3, 4:] = float("nan")
    z[4] = float("nan")
    z[5, ::2] = float("nan")
    z[6, 3], z[6, 30] = float("inf"), float("nan")
    z[7, 40:] = float("inf")
    z[8, :30], z[8, 40] = float("-inf"), float("nan")
    bias = 2 * _randn(5, E) if biased else None
    if biased:
        bias[7], bias[9] = 50.0, -50.0
    for groups, kept in ((1, 1), (4, 2), (8, 3)):
        for k in (1, 5, 12):
            got = mlxq.route_experts(z.cuda(), k, scoring, bias=None if bias is None else bias.cuda(), groups=groups, kept_groups=kept, group_best=best)
            ids, w = ref.route(z, k, scoring, bias=bias, groups=groups, kept=kept, best=best)
            if scoring == "softmax":
                for t in range(14):
                    if not bool((z[t] < float("inf")).all()):
                        ids[t] = torch.tensor(_undefined_choice(z[t].tolist(), k, groups, kept), dtype=torch.int32)
            banner("route_experts", scoring, biased, best, groups, kept, k)
            assert torch.equal(got.ids.cpu(), ids)
            g = got.weights.cpu().double()
            assert torch.equal(g.isnan(), w.isnan()) and ((g - w).abs() <= (2.0 ** -24 + 2.0 ** -40) * w.abs() + 2.0 ** -149)[~w.isnan()].all()
            starts, rows = ref.plan(ids, E)
            assert torch.equal(got.starts.cpu(), starts) and torch.equal(got.rows.cpu(), rows)
