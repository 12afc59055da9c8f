"""rotary, cache_append and copy_pages against their definitions (paged_ref), on the GPU."""
import math

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


def _table(n, R, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(n, R // 2, generator=g, dtype=torch.float64) * 6.3
    return torch.stack([a.cos(), a.sin()], -1).float()


def _x(seed, *shape, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,H,D,R", [(1, 1, 8, 8), (3, 5, 128, 128), (17, 2, 96, 48), (5, 3, 80, 20), (2, 40, 64, 2), (9, 1, 256, 250),
                                     (300, 7, 64, 64), (33, 3, 24, 24)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(mlxq, dtype, T, H, D, R, interleaved, inverse):
    banner("rotary", dtype, T, H, D, R, interleaved, inverse)
    x, table = _x(T, T, H, D, dtype=dtype), _table(50, R)
    pos = torch.randint(0, 50, (T,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    y = mlxq.rotary(x.cuda(), pos.cuda(), table.cuda(), interleaved, inverse)
    want = ref.rotated(x, pos.tolist(), table, interleaved, inverse)
    assert y.dtype == dtype and (y.cpu().double() - want).abs().max() <= ref.rotation_bound(x, table, dtype)
    assert torch.equal(y.cpu()[..., R:], x[..., R:])


def test_rotary_inverse_is_the_gradient(mlxq):
    """f(x) = sum(w * rotary(x)): the formula's gradient, and central differences of f, which is linear in x, so
    that they are exact but for the rounding of f: 2^-24 of the sum of its terms at each end, over the step."""
    for inter in (False, True):
        x, w, table = _x(1, 3, 2, 16, dtype=F32), _x(2, 3, 2, 16, dtype=F32), _table(9, 12)
        pos = torch.tensor([4, 0, 8], dtype=torch.int32).cuda()
        f = lambda t: float((mlxq.rotary(t.cuda(), pos, table.cuda(), inter).cpu().double() * w.double()).sum())  # noqa: E731
        g = mlxq.rotary(w.cuda(), pos, table.cuda(), inter, inverse=True).cpu().double()
        want = ref.rotated(w, pos.tolist(), table, inter, True)
        assert (g - want).abs().max() <= ref.rotation_bound(w, table, F32)
        h = 0.5
        terms = float((w.double().abs().sum())) * 8.0
        for e in ((0, 0, 0), (1, 1, 5), (2, 0, 11), (1, 0, 15), (2, 1, 7)):
            up, dn = x.clone(), x.clone()
            up[e] += h
            dn[e] -= h
            slope = (f(up) - f(dn)) / (float(up[e]) - float(dn[e]))
            assert abs(slope - float(g[e])) <= 2 * terms * 4 * 2.0 ** -24 / (2 * h)


def test_rotary_strides_and_places(mlxq):
    """A slice of a projection, head-major and odd-strided inputs, in place, a result into a slice; positions
    outside the table give NaN in the turned features only."""
    banner("rotary strides")
    table, pos = _table(20, 32).cuda(), torch.tensor([3, 19, 0, 7, 7], dtype=torch.int32).cuda()
    big = _x(0, 5, 9, 64).cuda()
    x = big[:, 2:6]
    want = mlxq.rotary(x.contiguous(), pos, table)
    assert torch.equal(mlxq.rotary(x, pos, table), want)
    assert torch.equal(mlxq.rotary(x.transpose(0, 1).contiguous().transpose(0, 1), pos, table), want)
    odd = torch.empty(5, 4, 67, dtype=BF16, device="cuda")[:, :, :64].copy_(x)
    assert torch.equal(mlxq.rotary(odd, pos, table), want)
    keep = big.clone()
    got = mlxq.rotary(x, pos, table, out=x)
    assert got is x and torch.equal(big[:, 2:6], want)
    assert torch.equal(big[:, :2], keep[:, :2]) and torch.equal(big[:, 6:], keep[:, 6:])
    for bad in (-1, 20, 2 ** 31 - 1, -2 ** 31):
        pos[2] = bad
        for inter, R in ((False, 32), (True, 32), (False, 20), (True, 20)):
            y = mlxq.rotary(keep, pos, table[:, :R // 2].contiguous(), inter)
            assert y[2, :, :R].isnan().all() and torch.equal(y[2, :, R:], keep[2, :, R:])
            assert torch.isfinite(y[[0, 1, 3, 4]]).all()


def test_rotary_table_and_frequencies(mlxq):
    """Angles in 64 bits: a position of 10^7 is as exact as position 1 (both within a unit in the last place of f32)."""
    f, m = mlxq.rotary_frequencies(64, 10000.0, "yarn", 8.0, 4096)
    t = mlxq.rotary_table(300, f, m).cpu().double()
    a = torch.arange(300, dtype=torch.float64)[:, None] * f
    want = m * torch.stack([a.cos(), a.sin()], -1)
    assert (t - want).abs().max() <= 2.0 ** -24 * m
    f = torch.tensor([1.0], dtype=torch.float64)
    n = 10 ** 7 + 1
    last = mlxq.rotary_table(n, f)[-1, 0].cpu().double()
    assert abs(float(last[0]) - math.cos(1e7)) <= 2.0 ** -24 and abs(float(last[1]) - math.sin(1e7)) <= 2.0 ** -24


APPEND = [[(1, 1), (1, 16), (1, 17), (1, 40)], [(5, 5), (0, 7), (16, 48), (1, 33), (37, 90)], [(40, 40)], [(7, 23)]]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,R,heads,group,page", [(64, 64, 2, 3, 16), (96, 48, 1, 1, 32), (80, 20, 2, 2, 64), (16, 16, 3, 1, 16),
                                                  (256, 256, 1, 2, 16), (64, 0, 2, 2, 16)])
@pytest.mark.parametrize("lens", APPEND, ids=["step", "ragged", "chunk", "inside"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_cache_append(mlxq, dtype, D, R, heads, group, page, lens, interleaved):
    """New tokens at every offset of a block: exactly their places change, keys turned by their places."""
    banner("cache_append", dtype, D, R, heads, group, page, lens, interleaved)
    pr = ref.Problem(D + R, lens, heads, group, D, page, dtype)
    before = [t.clone() for t in pr.cache("cpu")]
    table = _table(100, R) if R else None
    new_k = torch.cat([k[L - n:] for k, (n, L) in zip(pr.k, lens)])
    new_v = torch.cat([v[L - n:] for v, (n, L) in zip(pr.v, lens)])
    pos = [L - n + i for n, L in lens for i in range(n)]
    # the cache before the step: the new tokens' places hold something else
    old = ref.Problem(D + R + 1, lens, heads, group, D, page, dtype)
    for b, (n, L) in enumerate(lens):
        old.k[b][:L - n], old.v[b][:L - n] = pr.k[b][:L - n], pr.v[b][:L - n]
    old.pages = pr.pages
    k, v = old.cache()
    q = mlxq.cache_append(new_k.cuda(), new_v.cuda(), k, v, pr.batch(), q=pr.q.cuda(), table=table.cuda() if R else None,
                          interleaved=interleaved)
    turn = (lambda x: ref.rotated(x, pos, table, interleaved)) if R else (lambda x: x.double())
    bound = (lambda x: ref.rotation_bound(x, table, dtype)) if R else (lambda x: 0.0)
    assert (q.cpu().double() - turn(pr.q)).abs().max() <= bound(pr.q)
    want = turn(new_k)
    C = ref.pieces(dtype)
    kc, t = k.cpu(), 0
    for b, (n, L) in enumerate(lens):
        for p in range(L - n, L):
            at = pr.pages[b][p // page], p % page
            got = kc[at[0], :, at[1] // 16, :, at[1] % 16]
            assert (got.reshape(heads, D).double() - want[t]).abs().max() <= bound(new_k)
            kc[at[0], :, at[1] // 16, :, at[1] % 16] = pr.k[b][p].view(heads, D // C, C)
            t += 1
    as_bits = lambda x: x.view(torch.int16 if x.element_size() == 2 else torch.int32)  # noqa: E731
    assert torch.equal(as_bits(kc), as_bits(before[0])) and torch.equal(as_bits(v.cpu()), as_bits(before[1]))


def test_cache_append_positions_strides_and_places(mlxq):
    """Positions of the caller's, slices of one projection, queries in place, keys alone; tokens without a page or a
    place are not written and their neighbours are."""
    banner("cache_append places")
    lens = [(3, 20), (2, 35)]
    pr = ref.Problem(1, lens, 2, 2, 64)
    table, pos = _table(60, 64), torch.tensor([50, 0, 7, 59, 3], dtype=torch.int32)
    qkv = _x(3, 5, 8, 64).cuda()
    want_q, want_k = (mlxq.rotary(t.contiguous(), pos.cuda(), table.cuda()) for t in (qkv[:, :4], qkv[:, 4:6]))
    k, v = pr.cache()
    b = pr.batch()
    got = mlxq.cache_append(qkv[:, 4:6], qkv[:, 6:], k, v, b, q=qkv[:, :4], table=table.cuda(), positions=pos.cuda())
    assert torch.equal(got, want_q)
    kt, vt = mlxq.cache_tokens(k, v, pr.pages[0], 20)
    assert torch.equal(kt[17:], want_k[:3]) and torch.equal(vt[17:], qkv[:3, 6:])
    kt, vt = mlxq.cache_tokens(k, v, pr.pages[1], 35)
    assert torch.equal(kt[33:], want_k[3:]) and torch.equal(vt[33:], qkv[3:, 6:]) and torch.equal(kt[:33].cpu(), pr.k[1][:33])
    k1, v1 = pr.cache()
    q2 = qkv[:, :4].clone()
    assert mlxq.cache_append(qkv[:, 4:6], qkv[:, 6:], k1, v1, b, q=q2, table=table.cuda(), positions=pos.cuda(), out=q2) is q2
    assert torch.equal(q2, want_q)
    k2, v2 = pr.cache()
    assert mlxq.cache_append(qkv[:, 4:6], qkv[:, 6:], k2, v2, b, table=table.cuda(), positions=pos.cuda()) is None
    eq = lambda x, y: torch.equal(x.view(torch.int16), y.view(torch.int16))  # noqa: E731
    assert eq(k1, k) and eq(k2, k) and eq(v1, v) and eq(v2, v)
    # a page that is none, and more new tokens than the sequence has places
    k3, v3 = pr.cache()
    b = pr.batch()
    b.block_tables[0, 1], b.kv_lens[1] = 10 ** 8, 1
    mlxq.cache_append(qkv[:, 4:6], qkv[:, 6:], k3, v3, b, table=table.cuda(), positions=pos.cuda())
    k0, v0 = pr.cache()
    p = pr.pages[1][0]
    assert torch.equal(k3[p, :, 0, :, 0].reshape(2, 64), want_k[4]) and torch.equal(v3[p, :, 0, :, 0], qkv[4, 6:])
    k0[p, :, 0, :, 0], v0[p, :, 0, :, 0] = k3[p, :, 0, :, 0], v3[p, :, 0, :, 0]
    assert eq(k3, k0) and eq(v3, v0)


@pytest.mark.parametrize("shape,dim,dtype", [((3, 9, 2, 1, 8, 16, 8), None, BF16), ((9, 2, 4, 64, 4), None, F32), ((40, 1, 2, 4, 16, 8), None, F16),
                                             ((2, 2, 30, 1, 8, 128, 8), 2, BF16), ((4, 9, 2, 2, 16, 8), 1, BF16)])
def test_copy_pages(mlxq, shape, dim, dtype):
    banner("copy_pages", shape, dim)
    at = max(len(shape) - 6, 0) if dim is None else dim
    n = shape[at]
    cache = _x(0, *shape, dtype=dtype).cuda()
    order = torch.randperm(n, generator=torch.Generator().manual_seed(2)).int()
    src, dst = order[:n // 3].cuda(), order[n // 3:2 * (n // 3)].cuda()
    want = cache.clone()
    want.index_copy_(at, dst.long(), want.index_select(at, src.long()))
    tables = torch.randint(-2, n, (5, 37), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
    to = {s: d for s, d in zip(src.tolist(), dst.tolist())}
    want_t = torch.tensor([[to.get(e, e) for e in row] for row in tables.tolist()], dtype=torch.int32)
    wide = torch.full((5, 50), 3, dtype=torch.int32, device="cuda")
    wide[:, 4:41] = tables
    mlxq.copy_pages(cache, src, dst, wide[:, 4:41], dim=dim)
    assert torch.equal(cache, want) and torch.equal(wide[:, 4:41].cpu(), want_t)
    assert (wide[:, :4] == 3).all() and (wide[:, 41:] == 3).all()
    # ids outside the pool are left out, their entries too; nothing to copy is nothing
    bad = torch.tensor([0, -1, n, 2 ** 31 - 1], dtype=torch.int32).cuda()
    t = bad.clone().view(1, 4)
    mlxq.copy_pages(cache, bad, bad.flip(0).contiguous(), t, dim=dim)
    mlxq.copy_pages(cache, bad[:0], bad[:0], t, dim=dim)
    assert torch.equal(cache, want) and torch.equal(t[0], bad)


def test_copy_pages_many_moves(mlxq):
    """More moves than a workgroup stages at a time, offsets past 32 bits."""
    banner("copy_pages many")
    pool = 2 ** 33 // (16 * 64 * 2) + 3000
    cache = torch.empty((pool, 1, 1, 8, 16, 8), dtype=BF16, device="cuda")
    src = torch.arange(2500, dtype=torch.int32, device="cuda")
    dst = (pool - 1 - src).int()
    cache[:2500] = _x(0, 2500, 1, 1, 8, 16, 8).cuda()
    tables = torch.arange(3000, dtype=torch.int32, device="cuda").view(30, 100)
    mlxq.copy_pages(cache, src, dst, tables)
    assert torch.equal(cache[pool - 2500:].flip(0), cache[:2500])
    assert torch.equal(tables.view(-1)[:2500], dst) and torch.equal(tables.view(-1)[2500:].cpu(), torch.arange(2500, 3000).int())


def test_general_path_agrees(mlxq, monkeypatch):
    pr = ref.Problem(1, [(3, 20), (20, 35)], 2, 2, 64)
    table = _table(60, 64).cuda()
    x = _x(1, 23, 2, 64).cuda()
    pool = _x(2, 6, 2, 1, 8, 16, 8).cuda()
    move = torch.tensor([1, 4], dtype=torch.int32).cuda()

    def every():
        k, v = pr.cache()
        q = mlxq.cache_append(x, x, k, v, pr.batch(), q=pr.q.cuda(), table=table)
        p = pool.clone()
        mlxq.copy_pages(p, move, move + 1)
        return q, torch.nan_to_num(k), torch.nan_to_num(v), p, mlxq.rotary(x, torch.arange(23).int().cuda(), table, True, True)
    want = every()
    monkeypatch.setattr(mlxq._lib, "_fast", mlxq._lib._NoFast())
    for a, b in zip(every(), want):
        assert torch.equal(a, b)


def test_refusals(mlxq):
    pr = ref.Problem(2, [(3, 40)], 2, 2, 64)
    (k, v), b = pr.cache(), pr.batch()
    x, t = _x(1, 3, 2, 64).cuda(), _table(9, 64).cuda()
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")

    def refused(msg, f, *args, **kw):
        with pytest.raises(mlxq.MlxqError, match=msg) as e:
            f(*args, **kw)
        assert e.value.status in (1, 2)
    refused("positions", mlxq.rotary, x, pos[:2], t)
    refused("positions", mlxq.rotary, x, pos.long(), t)
    refused("table", mlxq.rotary, x, pos, t.double())
    refused("table", mlxq.rotary, x, pos, None)
    refused("rotary_dim", mlxq.rotary, x[..., :32], pos, t)
    refused("head_dim", mlxq.rotary, x[..., :4].contiguous(), pos, t[:, :2])
    refused("out", mlxq.rotary, x, pos, t, out=torch.empty(3, 2, 32, dtype=BF16, device="cuda"))
    refused("overlap", mlxq.rotary, x, pos, t, out=torch.empty(1, 2, 64, dtype=BF16, device="cuda").expand(3, 2, 64))
    refused("same strides", mlxq.rotary, x, pos, t, out=x.view(2, 3, 64).transpose(0, 1))
    refused("does not fit", mlxq.cache_append, x[:, :1], x, k, v, b)
    refused("does not fit", mlxq.cache_append, x, x[:2], k, v, b)
    refused("bfloat16", mlxq.cache_append, x.float(), x, k, v, b)
    refused("out without q", mlxq.cache_append, x, x, k, v, b, out=x)
    refused("query heads", mlxq.cache_append, x, x, k, v, b, q=_x(1, 3, 3, 64).cuda())
    refused("16 up to 256", mlxq.cache_append, _x(1, 3, 2, 8).cuda(), _x(1, 3, 2, 8).cuda(), k[:, :, :, :1].contiguous(), v[:, :, :, :8].contiguous(), b)
    refused("src|dst", mlxq.copy_pages, k, pos, pos[:2])
    refused("contiguous", mlxq.copy_pages, k[:, :1], pos, pos)
    refused("block_tables", mlxq.copy_pages, k, pos, pos, pos)


def test_paged_cache_end_to_end(mlxq):
    """Prompts, steps, forks, truncation and compaction through PagedCache, attention after each against the tokens
    that the sequences hold."""
    banner("PagedCache")
    heads, group, D, layers = 2, 2, 64, 2
    cache = mlxq.PagedCache(layers, 24, heads, D)
    cache.pool.fill_(math.nan)
    g = torch.Generator().manual_seed(4)
    book = {}

    def step(seqs, new):
        T = sum(new)
        b = cache.batch(seqs, new)
        for layer in range(layers):
            k, v, q = (torch.randn(T, h, D, generator=g).to(BF16) for h in (heads, heads, heads * group))
            t = 0
            for s, n in zip(seqs, new):
                kb, vb = book.setdefault((layer, s), (torch.empty(0, heads, D, dtype=BF16),) * 2)
                book[layer, s] = torch.cat([kb, k[t:t + n]]), torch.cat([vb, v[t:t + n]])
                t += n
            kc, vc = cache.layer(layer)
            mlxq.cache_append(k.cuda(), v.cuda(), kc, vc, b)
            got = mlxq.paged_attention(q.cuda(), kc, vc, b)
            pr = ref.Problem(0, [(n, cache.length(s)) for s, n in zip(seqs, new)], heads, group, D)
            pr.q, pr.k, pr.v = q, [book[layer, s][0] for s in seqs], [book[layer, s][1] for s in seqs]
            want, tol = ref.attention(pr)
            assert ((got.cpu().double() - want).abs() <= tol).all()
        return b

    a, b = cache.new(), cache.new()
    step([a, b], [37, 5])
    step([b, a], [1, 1])
    c, d = cache.fork([a, b])
    for layer in range(layers):
        book[layer, c], book[layer, d] = book[layer, a], book[layer, b]
    assert cache.pages_of(c)[:2] == cache.pages_of(a)[:2] and cache.pages_of(c)[2] != cache.pages_of(a)[2]
    step([a, b, c, d], [1, 2, 3, 12])
    cache.truncate(c, 20)
    for layer in range(layers):
        book[layer, c] = tuple(t[:20] for t in book[layer, c])
    step([c, a], [4, 1])
    cache.free(b)
    step([d, c], [20, 1])
    cache.free(a)
    used = cache.compact()
    assert used == 24 - cache.free_pages and all(p < used for s in (c, d) for p in cache.pages_of(s))
    step([c, d], [1, 1])
    tables = cache.batch([c, d], [0, 0]).block_tables
    cache.free(c)
    rows = tables[1:].clone()
    cache.compact(rows)
    n = len(cache.pages_of(d))
    assert rows[0, :n].tolist() == cache.pages_of(d) and (rows[0, n:] == -1).all()
    step([d], [3])
