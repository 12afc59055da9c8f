"""paged_attention against its definition in 64 bits (paged_ref): types, head widths, groups, page sizes, lengths
from none to several tiles, every option, and the places where it can go wrong: rows that see nothing, NaN
and infinities in hidden places, tables that name nothing, offsets past 32 bits, other streams and graphs."""
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


def _check(pr, got, opts, what=""):
    want, tol = ref.attention(pr, **opts)
    d = (got.double().cpu() - want).abs()
    worst = float((d / (tol + 1e-30)).max()) if d.numel() else 0.0
    print(f"    {what} error / bound {worst:.3f}", flush=True)
    assert got.dtype == pr.dtype and torch.isfinite(got).all()
    assert (d <= tol).all(), f"{what}: {worst:.3f} times the bound"


def _gpu(opts):
    """The reference's options as the framework takes them."""
    names = {"prefix": "prefix_lens", "slopes": "alibi_slopes"}
    return {names.get(k, k): v.cuda() if isinstance(v, torch.Tensor) else v for k, v in opts.items()}


# (new, cached) of each sequence: single tokens, odd lengths around blocks of 16 and 32, nothing new, chunks.
STEP = [(1, 1), (1, 15), (1, 16), (1, 17), (1, 31), (1, 33), (1, 200)]
DRAFT = [(4, 4), (3, 47), (0, 20), (5, 64), (2, 129)]
CHUNK = [(37, 37), (0, 0), (1, 70), (50, 131), (17, 300)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,group,heads,page", [(128, 4, 2, 16), (64, 8, 1, 32), (80, 1, 3, 64), (16, 3, 2, 16), (256, 2, 1, 128),
                                                (96, 7, 2, 16), (144, 1, 1, 16), (48, 20, 1, 1024)])
@pytest.mark.parametrize("lens", [STEP, DRAFT, CHUNK], ids=["step", "draft", "chunk"])
def test_lengths_and_shapes(mlxq, dtype, D, group, heads, page, lens):
    banner("paged_attention", dtype, D, group, heads, page, lens)
    pr = ref.Problem(D + group, lens, heads, group, D, page, dtype)
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch())
    _check(pr, got, {})


OPTIONS = {
    "window": dict(window=20),
    "window 1": dict(window=1),
    "wide window": dict(window=10 ** 6),
    "not causal": dict(causal=False),
    "not causal, window": dict(causal=False, window=9),
    "scale": dict(scale=0.5),
    "cap": dict(softcap=5.0),
    "prefix": dict(prefix=torch.tensor([3, 1000, 0, 64, 17], dtype=torch.int32)),
    "prefix, window": dict(prefix=torch.tensor([30, 0, 70, 90, 5], dtype=torch.int32), window=33),
    "bias": dict(slopes=torch.tensor([0.5, 0.0, 0.01, 0.1, 0.25, 1.0])),
    "sinks": dict(sinks=torch.tensor([0.0, 3.0, -2.0, 60.0, -math.inf, 1.0])),
    "all": dict(softcap=8.0, prefix=torch.tensor([3, 0, 0, 64, 17], dtype=torch.int32), window=50,
                slopes=torch.tensor([0.5, 0.0, 0.01, 0.1, 0.25, 1.0]), sinks=torch.tensor([0.0, 3.0, -2.0, 9.0, 2.0, 1.0])),
}


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("name", OPTIONS)
@pytest.mark.parametrize("lens", [DRAFT, CHUNK], ids=["draft", "chunk"])
def test_options(mlxq, dtype, name, lens):
    banner("paged_attention", name, dtype, lens)
    opts = OPTIONS[name]
    pr = ref.Problem(5, lens, 2, 3, 64, 32, dtype)
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), **_gpu(opts))
    _check(pr, got, opts, name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("new,opts", [(1, {}), (1, dict(window=700)), (6, dict(sinks=torch.tensor([1.0, -1.0]))),
                                      (40, dict(softcap=10.0))], ids=["one", "window", "sinks", "cap"])
def test_split_sequences(mlxq, dtype, new, opts):
    """Long sequences of very different lengths, cut over workgroups whose results are joined."""
    banner("paged_attention split", dtype, new, list(opts))
    pr = ref.Problem(new, [(new, 3001), (new, new), (1, 513), (new, 1100)], 1, 2, 64, 16, dtype)
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), **_gpu(opts))
    _check(pr, got, opts)


@pytest.mark.parametrize("lens,hints", [(DRAFT, (1, 1)), (CHUNK, (1, 1)), (CHUNK, (0, 0)), (STEP, (500, 10 ** 6)),
                                        ([(3, 2500)], (3, 100))])
def test_hints_change_nothing(mlxq, lens, hints):
    """max_q and max_kv plan the launch; lengths beyond or far below them give the same results."""
    banner("paged_attention hints", lens, hints)
    pr = ref.Problem(8, lens, 2, 4, 64)
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(max_q=hints[0], max_kv=hints[1], width=200))
    _check(pr, got, {})


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_see_nothing(mlxq, dtype):
    """More new tokens than the sequence has, and an empty sequence: zero rows, with and without sinks."""
    banner("paged_attention empty rows", dtype)
    pr = ref.Problem(3, [(5, 2), (2, 40), (3, 0)], 1, 2, 64, 16, dtype)
    for sinks in (None, torch.tensor([0.5, -0.5])):
        opts = {} if sinks is None else dict(sinks=sinks)
        got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), **_gpu(opts))
        _check(pr, got, opts)
        assert not got[:3].any() and got[3:7].any() and not got[7:].any()
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), causal=False)
    _check(pr, got, dict(causal=False))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("new,window", [(6, 0), (45, 0), (45, 11), (150, 0)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_hidden_values_do_not_reach_a_row(mlxq, dtype, new, window, value):
    """A token with a non-finite value: rows that do not see it are exact, rows that do carry it in that feature."""
    L = new + 37
    banner("paged_attention non-finite", dtype, new, window, value)
    pr = ref.Problem(new, [(new, L), (2, 30)], 1, 2, 64, 16, dtype)
    where = L - new // 2 - 1
    pr.v[0][where, 0, 5] = value
    clean = ref.Problem(new, [(new, L), (2, 30)], 1, 2, 64, 16, dtype)
    opts = dict(window=window) if window else {}
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), **opts).cpu()
    want, tol = ref.attention(clean, **opts)
    place = torch.arange(L - new, L)
    sees = (place >= where) & ((place < where + window) if window else torch.ones(new, dtype=torch.bool))
    assert sees.any() and not sees.all()
    sees = torch.cat([sees, torch.zeros(2, dtype=torch.bool)])
    hit = got[sees][:, :, 5]
    assert (hit == value).all() if not math.isnan(value) else hit.isnan().all()
    got = got.double()
    got[sees, :, 5] = want[sees, :, 5]
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_hidden_keys_do_not_reach_a_row(mlxq, dtype):
    banner("paged_attention NaN keys", dtype)
    pr = ref.Problem(1, [(70, 100)], 1, 2, 64, 16, dtype)
    pr.k[0][60:] = math.nan
    clean = ref.Problem(1, [(70, 100)], 1, 2, 64, 16, dtype)
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch()).cpu()
    want, tol = ref.attention(clean)
    assert ((got[:30].double() - want[:30]).abs() <= tol[:30]).all()
    assert got[30:].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("entry", [-1, 2 ** 31 - 1, 10 ** 6])
def test_tables_that_name_no_page(mlxq, dtype, new, entry):
    """An entry outside the pool is not followed: the rows that see it are NaN, all others exact."""
    banner("paged_attention bad page", dtype, new, entry)
    pr = ref.Problem(new, [(new, 150), (2, 70)], 2, 2, 64, 16, dtype)
    b = pr.batch()
    b.block_tables[0, 8] = entry  # tokens 128 .. 143
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), b).cpu()
    want, tol = ref.attention(pr)
    bad = torch.arange(pr.T) < new
    bad &= torch.cat([torch.arange(150 - new, 150), torch.zeros(2, dtype=torch.long)]) >= 128
    assert got[bad].isnan().all() and bad.any()
    assert ((got[~bad].double() - want[~bad]).abs() <= tol[~bad]).all()
    # pages before the window are never looked up
    b.block_tables[0, 8] = pr.pages[0][8]
    b.block_tables[0, :2] = entry
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), b, window=40)
    if new == 1:
        _check(pr, got, dict(window=40))


@pytest.mark.parametrize("new", [1, 40])
def test_strides(mlxq, new):
    """Queries as a slice of a projection or head-major, a result into a wider tensor, pages of a wider pool, tables
    of a wider table."""
    banner("paged_attention strides", new)
    pr = ref.Problem(4, [(new, 77), (2, 50)], 2, 2, 64)
    want = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch())
    _check(pr, want, {})
    k, v = pr.cache()
    wide = torch.full((pr.T, 9, 64), math.nan, dtype=BF16, device="cuda")
    wide[:, 3:7] = pr.q.cuda()
    assert torch.equal(mlxq.paged_attention(wide[:, 3:7], k, v, pr.batch()), want)
    major = pr.q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(mlxq.paged_attention(major, k, v, pr.batch()), want)
    odd = torch.empty(pr.T, 4, 65, dtype=BF16, device="cuda")[:, :, :64].copy_(pr.q.cuda())
    assert torch.equal(mlxq.paged_attention(odd, k, v, pr.batch()), want)
    out = torch.zeros_like(wide)
    got = mlxq.paged_attention(pr.q.cuda(), k, v, pr.batch(), out=out[:, 1:5])
    assert got.data_ptr() == out[:, 1:5].data_ptr() and torch.equal(out[:, 1:5], want)
    assert not out[:, 0].any() and not out[:, 5:].any()
    kk = torch.full((k.shape[0], 2, *k.shape[1:]), math.nan, dtype=BF16, device="cuda")
    vv = torch.full((v.shape[0], 3, *v.shape[1:]), math.nan, dtype=BF16, device="cuda")
    kk[:, 1], vv[:, 1] = k, v
    assert torch.equal(mlxq.paged_attention(pr.q.cuda(), kk[:, 1], vv[:, 1], pr.batch()), want)
    b = pr.batch()
    t = torch.full((2, 40), -7, dtype=torch.int32, device="cuda")
    t[:, 3:3 + b.block_tables.shape[1]] = b.block_tables
    view = b._replace(block_tables=t[:, 3:3 + b.block_tables.shape[1]])
    assert torch.equal(mlxq.paged_attention(pr.q.cuda(), k, v, view), want)


def test_tokens_outside_every_sequence_are_left_alone(mlxq):
    """A step padded to a fixed number of tokens: rows before the first and after the last sequence keep out's."""
    banner("paged_attention padding rows")
    for lens in ([(1, 900), (1, 20)], [(30, 90), (1, 2000)]):
        pr = ref.Problem(2, lens, 1, 2, 64)
        n = pr.T
        q = torch.full((n + 5, 2, 64), math.nan, dtype=BF16, device="cuda")
        q[2:2 + n] = pr.q.cuda()
        b = pr.batch()
        out = torch.full_like(q, 7.0)
        mlxq.paged_attention(q, *pr.cache(), b._replace(q_starts=b.q_starts + 2), out=out)
        _check(pr, out[2:2 + n], {})
        assert (out[:2] == 7).all() and (out[2 + n:] == 7).all()


@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_32_bits(mlxq, new):
    """Pages whose first element lies past 2^32 elements into each pool."""
    banner("paged_attention long pool", new)
    pr = ref.Problem(6, [(new, 60)], 1, 2, 64)
    k, v = pr.cache()
    far = 2 ** 32 // (16 * 64) + 5
    kk, vv = (torch.empty((far + 4, *t.shape[1:]), dtype=BF16, device="cuda") for t in (k, v))
    at = torch.tensor([1, far, 3, far + 3], device="cuda")
    mine = torch.tensor(pr.pages[0], device="cuda")
    kk[at], vv[at] = k[mine], v[mine]
    b = pr.batch()
    b.block_tables[0] = at.int()
    _check(pr, mlxq.paged_attention(pr.q.cuda(), kk, vv, b), {})


@pytest.mark.parametrize("lens", [[(1, 3000), (1, 9)], [(60, 200), (1, 40)]], ids=["step", "chunk"])
def test_streams_and_graphs(mlxq, lens):
    """On a side stream; and captured, then replayed with other queries, lengths and tables, each replay against the
    eager result bit for bit."""
    banner("paged_attention graph", lens)
    pr = ref.Problem(11, lens, 1, 4, 64)
    k, v = pr.cache()
    q, b = pr.q.cuda(), pr.batch()
    want = mlxq.paged_attention(q, k, v, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mlxq.paged_attention(q, k, v, b)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlxq.paged_attention(q, k, v, b)
    g = torch.Generator(device="cuda").manual_seed(1)
    for rep in range(4):
        out.fill_(math.nan)
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        b.kv_lens[0] = lens[0][1] - 13 * rep
        b.block_tables[1, 0] = pr.pages[0][rep]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mlxq.paged_attention(q, k, v, b)), rep
    del graph


def test_same_result_every_time(mlxq):
    """Split sequences are joined in a fixed order."""
    banner("paged_attention repeats")
    pr = ref.Problem(2, [(1, 4000), (3, 2222)], 2, 2, 64)
    q, (k, v), b = pr.q.cuda(), pr.cache(), pr.batch()
    want = mlxq.paged_attention(q, k, v, b)
    for _ in range(20):
        assert torch.equal(mlxq.paged_attention(q, k, v, b), want)


def test_empty_steps(mlxq):
    pr = ref.Problem(2, [(1, 40)], 1, 2, 64)
    k, v = pr.cache()
    b = pr.batch()
    q = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
    assert mlxq.paged_attention(q, k, v, b).shape == (0, 2, 64)
    none = mlxq.CacheBatch(b.block_tables[:0], b.q_starts[:1], b.kv_lens[:0], 0, 0)
    assert mlxq.paged_attention(q, k, v, none).shape == (0, 2, 64)


def test_general_path_agrees(mlxq, monkeypatch):
    """The calls through ctypes give what the native call path gives."""
    pr = ref.Problem(2, CHUNK, 2, 3, 64)
    q, (k, v), b = pr.q.cuda(), pr.cache(), pr.batch()
    opts = _gpu(OPTIONS["all"])
    want = mlxq.paged_attention(q, k, v, b, **opts)
    monkeypatch.setattr(mlxq._lib, "_fast", mlxq._lib._NoFast())
    assert torch.equal(mlxq.paged_attention(q, k, v, b, **opts), want)


def test_refusals(mlxq):
    pr = ref.Problem(2, [(3, 40)], 2, 2, 64)
    q, (k, v), b = pr.q.cuda(), pr.cache(), pr.batch()
    f = mlxq.paged_attention

    def refused(msg, *args, **kw):
        with pytest.raises(mlxq.MlxqError, match=msg) as e:
            f(*args, **kw)
        assert e.value.status == 1
    refused("dtype|bfloat16", q.float(), k, v, b)
    refused("does not fit", q[:, :3], k, v, b)
    refused("does not fit", q[:, :, :32], k, v, b)
    refused("must be", q[0], k, v, b)
    refused("k_cache", q, k[0], v, b)
    refused("v_cache", q, k, v[:, :1], b)
    refused("contiguous", q, k[:, :, :, ::2], v[:, :, :, ::2], b)
    refused("block_tables", q, k, v, b._replace(block_tables=b.block_tables.long()))
    refused("q_starts", q, k, v, b._replace(q_starts=b.q_starts[:1]))
    refused("kv_lens", q, k, v, b._replace(kv_lens=b.kv_lens.cpu()))
    refused("scale", q, k, v, b, scale=0.0)
    refused("scale", q, k, v, b, scale=math.inf)
    refused("softcap", q, k, v, b, softcap=-1.0)
    refused("window", q, k, v, b, window=-1)
    refused("prefix_lens", q, k, v, b, prefix_lens=torch.zeros(2, dtype=torch.int32, device="cuda"))
    refused("alibi_slopes", q, k, v, b, alibi_slopes=torch.zeros(2, device="cuda"))
    refused("sinks", q, k, v, b, sinks=torch.zeros(4, dtype=BF16, device="cuda"))
    refused("out", q, k, v, b, out=torch.empty(3, 4, 64, device="cuda"))
    refused("overlap", q, k, v, b, out=torch.empty(1, 4, 64, dtype=BF16, device="cuda").expand(3, 4, 64))
