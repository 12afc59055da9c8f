"""Block tables narrower than their sequences: a token past the table has no page, as one whose entry names none.  It is not
written (and no other token in its place), rows that see it are NaN, and all others are what they are with the whole table."""
import pytest
import torch

import paged_ref as ref
from gpu_util import banner

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mlxq():
    import mlxq as m
    m.load()
    return m


def _cut(b, width):
    return b._replace(block_tables=b.block_tables[:, :width].contiguous())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,width", [([(1, 33), (1, 20)], 2), ([(3, 40), (2, 18)], 2), ([(12, 40), (1, 32)], 2), ([(40, 40), (5, 70)], 1),
                                        ([(4, 40), (2, 9)], 0)])
def test_append(mlxq, dtype, lens, width):
    banner("cache_append narrow", dtype, lens, width)
    pr = ref.Problem(3, lens, 2, 2, 64, 16, dtype)
    a = torch.rand(100, 32, generator=torch.Generator().manual_seed(0), dtype=torch.float64) * 6.3
    table = torch.stack([a.cos(), a.sin()], -1).float().cuda()
    new_k = torch.cat([k[L - n:] for k, (n, L) in zip(pr.k, lens)]).cuda()
    new_v = torch.cat([v[L - n:] for v, (n, L) in zip(pr.v, lens)]).cuda()
    k, v = pr.cache()
    want_k, want_v = k.clone(), v.clone()
    mlxq.cache_append(new_k + 1, new_v + 1, want_k, want_v, pr.batch(), table=table)
    cut = [t.clone() for t in (k, v)]
    q = mlxq.cache_append(new_k + 1, new_v + 1, *cut, _cut(pr.batch(), width), q=pr.q.cuda(), table=table)
    pos = torch.tensor([L - n + i for n, L in lens for i in range(n)], dtype=torch.int32, device="cuda")
    assert torch.equal(q, mlxq.rotary(pr.q.cuda(), pos, table))
    # what the table names is as with the whole one, all else as before
    eq = lambda x, y: torch.equal(x.view(torch.uint8), y.view(torch.uint8))  # noqa: E731
    named = torch.zeros(k.shape[0], dtype=torch.bool)
    for pages in pr.pages:
        named[pages[:width]] = True
    for got, whole, before in zip(cut, (want_k, want_v), (k, v)):
        assert eq(got[named], whole[named]) and eq(got[~named], before[~named])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lens,width", [([(1, 33), (1, 20)], 2), ([(1, 33), (1, 32)], 0), ([(5, 40), (2, 18)], 2), ([(60, 100), (1, 70), (3, 17)], 5),
                                        ([(130, 400), (1, 900)], 18), ([(2, 3000), (1, 1500), (1, 40)], 150)])
@pytest.mark.parametrize("opts", [{}, dict(window=25), dict(causal=False), dict(prefix=[90, 0, 3])], ids=["causal", "window", "all", "prefix"])
def test_attention(mlxq, dtype, lens, width, opts):
    banner("paged_attention narrow", dtype, lens, width, opts)
    opts = dict(opts)
    if "prefix" in opts:
        opts["prefix"] = torch.tensor(opts["prefix"][:len(lens)], dtype=torch.int32)
    pr = ref.Problem(4, lens, 1, 2, 64, 16, dtype)
    given = {{"prefix": "prefix_lens"}.get(n, n): v.cuda() if isinstance(v, torch.Tensor) else v for n, v in opts.items()}
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), _cut(pr.batch(), width), **given).cpu()
    want, tol = ref.attention(pr, **opts)
    t = 0
    for b, (n, L) in enumerate(lens):
        for p in range(L - n, L):
            upto = L if opts.get("causal") is False else min(L, max(p + 1, int(opts["prefix"][b]) if "prefix" in opts else 0))
            if upto > 16 * width:
                assert got[t].isnan().all(), (b, p)
            else:
                assert ((got[t].double() - want[t]).abs() <= tol[t]).all(), (b, p)
            t += 1


def test_the_longest_lengths(mlxq):
    """Lengths up to the largest integer: nothing is written or read, rows are NaN."""
    banner("paged cache, largest lengths")
    for new in (1, 40):
        for L in (2 ** 30 - 1, 2 ** 30, 2 ** 30 + 5, 2 ** 31 - 1):
            pr = ref.Problem(4, [(new, 64)], 1, 2, 64)
            k, v = pr.cache()
            b = pr.batch()
            b.kv_lens[0] = L
            before = k.clone(), v.clone()
            mlxq.cache_append(pr.k[0][:new].cuda(), pr.v[0][:new].cuda(), k, v, b)
            assert torch.equal(k.view(torch.int16), before[0].view(torch.int16)) and torch.equal(v.view(torch.int16), before[1].view(torch.int16))
            assert mlxq.paged_attention(pr.q.cuda(), k, v, b).isnan().all()
            assert mlxq.paged_attention(pr.q.cuda(), k, v, b, window=20).isnan().all()
