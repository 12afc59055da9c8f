"""paged_attention over several tiles of rows and keys: scores whose maximum keeps rising, non-finite values in tiles that
some rows do not see, wide heads, split chunks, workspaces with arbitrary contents, drawn shapes.  Bounds: paged_ref."""
import ctypes
import math
import random

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


def _check(got, want, tol):
    d = (got.double().cpu() - want).abs()
    print(f"    error / bound {float((d / (tol + 1e-30)).max()):.3f}", flush=True)
    assert torch.isfinite(got).all() and (d <= tol).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("opts", [{}, dict(softcap=30.0), dict(window=150, slopes=torch.tensor([0.1, 0.02]))],
                         ids=["plain", "cap", "bias"])
def test_rising_scores(mlxq, dtype, D, opts):
    """Keys grow along the sequence, so that later tiles hold far larger scores than the ones before them."""
    banner("paged_attention rising", dtype, D, list(opts))
    pr = ref.Problem(D, [(70, 500), (3, 260)], 1, 2, D, 16, dtype, std=1.0)
    for k in pr.k:
        k *= torch.linspace(0.0, 8.0, k.shape[0]).view(-1, 1, 1).to(dtype)
    given = {{"slopes": "alibi_slopes"}.get(n, n): v.cuda() if isinstance(v, torch.Tensor) else v for n, v in opts.items()}
    _check(mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), **given), *ref.attention(pr, **opts))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [128, 192, 256])
@pytest.mark.parametrize("window", [0, 40])
def test_non_finite_values_in_part_seen_tiles(mlxq, dtype, D, window):
    """Three tokens of one tile hold +inf, -inf and NaN in features of different lanes: rows that see none are exact,
    the others exact in all other features."""
    new, L = 90, 400
    banner("paged_attention non-finite", dtype, D, window)
    lens = [(new, L), (3, 30)]
    pr, clean = (ref.Problem(D, lens, 1, 2, D, 32, dtype) for _ in range(2))
    bad = {L - 50: (7, math.inf), L - 40: (D - 1, -math.inf), L - 30: (D // 2 + 3, math.nan)}
    for j, (d, x) in bad.items():
        pr.v[0][j, 0, d] = x
    opts = dict(window=window) if window else {}
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), **opts).cpu()
    want, tol = ref.attention(clean, **opts)
    place = torch.arange(L - new, L)
    got = got.double()
    for j, (d, x) in bad.items():
        sees = torch.zeros(new + 3, dtype=torch.bool)
        sees[:new] = (place >= j) & ((place < j + window) if window else True)
        assert sees.any() and not sees.all()
        hit = got[sees][:, :, d]
        assert hit.isnan().all() if math.isnan(x) else (hit == x).all()
        got[sees, :, d] = want[sees, :, d]
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("D,dtype,new,length", [(128, BF16, 1, 3000), (256, F16, 130, 2500), (64, F32, 5, 2000)])
def test_workspace_contents_do_not_matter(mlxq, D, dtype, new, length):
    """The C entry with a workspace of all-ones bits (NaN, and the largest counts), of zeros, and of the smallest allowed size."""
    banner("paged_attention workspace", D, dtype, new, length)
    P = mlxq.paged
    pr = ref.Problem(D, [(new, length), (1, 700)], 2, 2, D, 16, dtype)
    q, (k, v), b = pr.q.cuda(), pr.cache(), pr.batch()
    want = mlxq.paged_attention(q, k, v, b)
    cache, (view, keep) = P._cache("test", k, v), P._batch("test", b, q.device)
    opts = P.Attention(1.0 / math.sqrt(D), 1, 0, 0.0, None, None, None)
    out = torch.empty_like(q)
    (_, qv), (_, ov) = P._heads("test", "q", q), P._heads("test", "out", out)
    lib, ref_of = mlxq.load(), ctypes.byref
    need = lib.mlxq_paged_attention_workspace_size(q.shape[0], 4, ref_of(cache), ref_of(view), ref_of(opts))
    assert need > 0
    for byte in (0xff, 0x00, 0x7f):
        ws = torch.full((need,), byte, dtype=torch.uint8, device="cuda")
        out.fill_(float("nan"))
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        rc = lib.mlxq_paged_attention(ref_of(qv), q.shape[0], ref_of(cache), ref_of(view), ref_of(opts), ref_of(ov),
                                      ctypes.c_void_p(ws.data_ptr()), need, stream)
        assert rc == 0 and torch.equal(out, want), byte
    rc = lib.mlxq_paged_attention(ref_of(qv), q.shape[0], ref_of(cache), ref_of(view), ref_of(opts), ref_of(ov),
                                  ctypes.c_void_p(ws.data_ptr()), need - 1, stream)
    assert rc == 1
    del keep


@pytest.mark.parametrize("seed", range(24))
def test_drawn_shapes(mlxq, seed):
    r = random.Random(900 + seed)
    dtype = r.choice([BF16, F16, F32])
    heads, group = r.choice([1, 1, 2, 3]), r.choice([1, 2, 3, 5, 8])
    D, page = 16 * r.randint(1, 16), r.choice([16, 32, 64, 256])
    lens = []
    for _ in range(r.randint(1, 5)):
        n = r.choice([0, 1, 1, 2, r.randint(3, 20), r.randint(20, 160)])
        n = min(n, 700 // (heads * group))
        lens.append((n, n + r.choice([0, r.randint(1, 40), r.randint(1, 900)])))
    opts = {}
    if r.random() < 0.4:
        opts["window"] = r.choice([1, 17, 200])
    if r.random() < 0.3:
        opts["softcap"] = r.choice([3.0, 50.0])
    if r.random() < 0.3:
        opts["causal"] = False
    if r.random() < 0.3:
        opts["prefix"] = torch.tensor([r.randint(0, 300) for _ in lens], dtype=torch.int32)
    if r.random() < 0.3:
        opts["slopes"] = torch.rand(heads * group, generator=torch.Generator().manual_seed(seed))
    if r.random() < 0.3:
        opts["sinks"] = torch.randn(heads * group, generator=torch.Generator().manual_seed(seed))
    banner("paged_attention drawn", seed, dtype, heads, group, D, page, lens, list(opts))
    pr = ref.Problem(seed, lens, heads, group, D, page, dtype)
    given = {{"slopes": "alibi_slopes", "prefix": "prefix_lens"}.get(n, n): v.cuda() if isinstance(v, torch.Tensor) else v
             for n, v in opts.items()}
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), **given)
    if pr.T:
        _check(got, *ref.attention(pr, **opts))
