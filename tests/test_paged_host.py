"""The paged-cache operators' host side, on the CPU: argument checks of the C ABI before any device work, the
frequencies' scalings against their formulas, and PagedCache's book-keeping."""
import ctypes
import math
import random

import pytest
import torch

import mlxq
from mlxq import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


P = 4096  # any aligned address: nothing below gets as far as reading it


def _cache(**kw):
    f = dict(k=P, v=P, k_page_stride=2048, v_page_stride=2048, pages=9, page_size=16, heads=2, head_dim=64, dtype=1)
    f.update(kw)
    return _lib.PagedCacheView(**f)


def _batch(**kw):
    f = dict(block_tables=P, q_starts=P, kv_lens=P, sequences=3, table_width=4, table_stride=4, max_q=1, max_kv=64)
    f.update(kw)
    return _lib.PagedBatch(**f)


def _heads(heads, **kw):
    f = dict(data=P, heads=heads, token_stride=64 * heads, head_stride=64)
    f.update(kw)
    return _lib.Heads(**f)


def _attn(**kw):
    f = dict(scale=0.125, causal=1, window=0, softcap=0.0, prefix_lens=None, alibi_slopes=None, sinks=None)
    f.update(kw)
    return _lib.Attention(**f)


def _r(x):
    return None if x is None else ctypes.byref(x)


@pytest.mark.parametrize("msg,kw", [
    ("q or out is null", dict(q=None)), ("cache is null", dict(cache=None)), ("batch is null", dict(batch=None)),
    ("options are null", dict(opts=None)), ("T=-1", dict(T=-1)),
    ("dtype 7", dict(cache=_cache(dtype=7))), ("page_size 24", dict(cache=_cache(page_size=24))),
    ("page_size 8", dict(cache=_cache(page_size=8))), ("2048", dict(cache=_cache(page_size=2048))),
    ("head_dim 72", dict(cache=_cache(head_dim=72))), ("head_dim 272", dict(cache=_cache(head_dim=272))),
    ("no pages", dict(cache=_cache(pages=0))), ("k cache is null", dict(cache=_cache(k=None))),
    ("v cache must be 16", dict(cache=_cache(v=P + 8))), ("page strides", dict(cache=_cache(k_page_stride=2047))),
    ("page strides", dict(cache=_cache(v_page_stride=2050))), ("0 heads", dict(cache=_cache(heads=0))),
    ("q_starts is null", dict(batch=_batch(q_starts=None))), ("kv_lens must be 4", dict(batch=_batch(kv_lens=P + 2))),
    ("block_tables is null", dict(batch=_batch(block_tables=None))), ("overlap", dict(batch=_batch(table_stride=3))),
    ("max_q and max_kv", dict(batch=_batch(max_q=-1))), ("block tables of", dict(batch=_batch(sequences=-2))),
    ("scale", dict(opts=_attn(scale=-1.0))), ("scale", dict(opts=_attn(scale=math.nan))),
    ("softcap", dict(opts=_attn(softcap=math.nan))), ("window", dict(opts=_attn(window=-3))),
    ("sinks must be 4", dict(opts=_attn(sinks=P + 1))), ("5 query heads over 2", dict(q=_heads(5), out=_heads(5))),
    ("q must be 16", dict(q=_heads(4, data=P + 2))), ("strides of q", dict(q=_heads(4, token_stride=251))),
    ("out overlap", dict(out=_heads(4, token_stride=0))), ("out overlap", dict(out=_heads(4, head_stride=32))),
    ("out overlap", dict(out=_heads(4, token_stride=128))), ("different heads", dict(out=_heads(2))),
])
def test_attention_refusals(lib, msg, kw):
    a = dict(q=_heads(4), T=3, cache=_cache(), batch=_batch(), opts=_attn(), out=_heads(4))
    a.update(kw)
    rc = lib.mlxq_paged_attention(_r(a["q"]), a["T"], _r(a["cache"]), _r(a["batch"]), _r(a["opts"]), _r(a["out"]), None, 0, None)
    assert rc in (_lib.MLXQ_EINVAL, _lib.MLXQ_EUNSUPPORTED) and msg in lib.mlxq_last_error().decode(), lib.mlxq_last_error()


def test_attention_workspace(lib):
    """A long sequence is split and needs a workspace, which is refused when absent, short or misaligned."""
    q, c, b, o = _heads(4), _cache(pages=10 ** 6), _batch(sequences=1, table_width=10 ** 5, table_stride=10 ** 5, max_kv=10 ** 6), _attn()
    need = lib.mlxq_paged_attention_workspace_size(1, 4, _r(c), _r(b), _r(o))
    assert need >= 4 * 64 * 4
    for ws, size in ((None, need), (P, need - 1), (P + 4, need)):
        assert lib.mlxq_paged_attention(_r(q), 1, _r(c), _r(b), _r(o), _r(q), ws, size, None) == _lib.MLXQ_EINVAL
        assert b"workspace" in lib.mlxq_last_error()
    assert lib.mlxq_paged_attention_workspace_size(1, 3, _r(c), _r(b), _r(o)) == 0  # refused arguments
    assert lib.mlxq_paged_attention_workspace_size(0, 4, _r(c), _r(b), _r(o)) == 0
    short = _batch(sequences=1, max_kv=40)
    assert lib.mlxq_paged_attention_workspace_size(1, 4, _r(c), _r(short), _r(o)) == 0


def test_empty_problems_are_no_ops(lib):
    q, none = _heads(4, data=None), _batch(sequences=0, q_starts=None, kv_lens=None, block_tables=None)
    assert lib.mlxq_paged_attention(_r(q), 0, _r(_cache()), _r(_batch()), _r(_attn()), _r(q), None, 0, None) == _lib.MLXQ_OK
    assert lib.mlxq_paged_attention(_r(q), 5, _r(_cache()), _r(none), _r(_attn()), _r(q), None, 0, None) == _lib.MLXQ_OK
    assert lib.mlxq_cache_append(_r(q), _r(q), 0, _r(_cache()), _r(_batch()), None, None, 0, 0, 0, None, None, None) == _lib.MLXQ_OK
    assert lib.mlxq_cache_copy_pages(None, 2, 4096, 9, 1024, 1024, None, None, 0, None, 0, 0, 0, None) == _lib.MLXQ_OK
    assert lib.mlxq_rotary(_r(q), 1, 0, 64, None, P, 9, 64, 0, 0, _r(q), None) == _lib.MLXQ_OK
    assert lib.mlxq_rotary_table((ctypes.c_double * 1)(1.0), 2, 1.0, 0, None, None) == _lib.MLXQ_OK


@pytest.mark.parametrize("msg,kw", [
    ("dtype", dict(dtype=3)), ("T=-4", dict(T=-4)), ("head_dim 60", dict(D=60)), ("rotary_dim 63", dict(R=63)),
    ("rotary_dim 66", dict(R=66)), ("rotary_dim is 0", dict(R=0)), ("rotary_dim 258", dict(R=258, D=512)), ("table", dict(table=P + 8)),
    ("table", dict(table=None)), ("table of 0", dict(rows=0)), ("x must be 16", dict(x=_heads(2, data=P + 4))), ("y is null", dict(y=None)),
    ("positions is null", dict(pos=None)), ("different heads", dict(y=_heads(3, data=2 * P))), ("overlap", dict(y=_heads(2, data=2 * P, token_stride=64))),
    ("same strides", dict(y=_heads(2, token_stride=256))),
])
def test_rotary_refusals(lib, msg, kw):
    a = dict(x=_heads(2), dtype=1, T=5, D=64, pos=P, table=P, rows=9, R=64, y=_heads(2, data=2 * P))
    a.update(kw)
    rc = lib.mlxq_rotary(_r(a["x"]), a["dtype"], a["T"], a["D"], a["pos"], a["table"], a["rows"], a["R"], 0, 0, _r(a["y"]), None)
    assert rc == _lib.MLXQ_EINVAL and msg in lib.mlxq_last_error().decode(), lib.mlxq_last_error()


@pytest.mark.parametrize("msg,kw", [
    ("cache is null", dict(cache=None)), ("k is null", dict(k=None)), ("cache's 2 heads", dict(v=_heads(3))), ("come together", dict(q=_heads(4))),
    ("query heads", dict(q=_heads(3), q_out=_heads(3))), ("query heads", dict(q=_heads(4), q_out=_heads(2, data=2 * P))), ("rotary_dim 80", dict(R=80)),
    ("overlap", dict(q=_heads(4), q_out=_heads(4, token_stride=0))), ("same strides", dict(q=_heads(4), q_out=_heads(4, token_stride=512))),
    ("positions must be 4", dict(pos=P + 1)),
])
def test_append_refusals(lib, msg, kw):
    a = dict(k=_heads(2), v=_heads(2), cache=_cache(), q=None, q_out=None, R=64, pos=None)
    a.update(kw)
    rc = lib.mlxq_cache_append(_r(a["k"]), _r(a["v"]), 3, _r(a["cache"]), _r(_batch()), a["pos"], P, 9, a["R"], 0, _r(a["q"]), _r(a["q_out"]), None)
    assert rc == _lib.MLXQ_EINVAL and msg in lib.mlxq_last_error().decode(), lib.mlxq_last_error()


@pytest.mark.parametrize("msg,kw", [
    ("count=-1", dict(count=-1)), ("multiples of 16", dict(page=1000)), ("multiples of 16", dict(stride=512)), ("planes overlap", dict(plane=512)),
    ("src is null", dict(src=None)), ("dst must be 4", dict(dst=P + 2)), ("cache must be 16", dict(cache=P + 8)), ("block tables", dict(width=9)),
    ("too large", dict(planes=2 ** 20, count=2 ** 20)),
])
def test_copy_refusals(lib, msg, kw):
    a = dict(cache=P, planes=2, plane=9 * 1024, page=1024, stride=1024, src=P, dst=P, count=3, width=4)
    a.update(kw)
    rc = lib.mlxq_cache_copy_pages(a["cache"], a["planes"], a["plane"], 9, a["page"], a["stride"], a["src"], a["dst"], a["count"], P, 2, a["width"], 4, None)
    assert rc == _lib.MLXQ_EINVAL and msg in lib.mlxq_last_error().decode(), lib.mlxq_last_error()


def _freqs(R, base=10000.0):
    return [base ** (-2 * i / R) for i in range(R // 2)]


def test_frequencies():
    """Each scaling against its formula, written out once more."""
    close = lambda a, b: all(abs(x - y) <= 1e-14 * y for x, y in zip(a, b)) and len(a) == len(b)  # noqa: E731
    f, m = mlxq.rotary_frequencies(64)
    assert m == 1.0 and f.dtype == torch.float64 and close(f.tolist(), _freqs(64))
    f, m = mlxq.rotary_frequencies(64, 500000.0, "linear", 4.0)
    assert m == 1.0 and close(f.tolist(), [x / 4 for x in _freqs(64, 500000.0)])
    f, m = mlxq.rotary_frequencies(64, 10000.0, "ntk", 8.0)
    assert m == 1.0 and close(f.tolist(), _freqs(64, 10000.0 * 8.0 ** (64 / 62)))
    assert close([float(f[-1])], [_freqs(64)[-1] / 8.0])  # the slowest pair is slowed by the factor
    turns = [8192 * x / (2 * math.pi) for x in _freqs(128, 500000.0)]
    f, m = mlxq.rotary_frequencies(128, 500000.0, "llama3", 8.0, 8192)
    want = []
    for n, x in zip(turns, _freqs(128, 500000.0)):
        s = min(max((n - 1) / 3, 0.0), 1.0)
        want.append((1 - s) * x / 8 + s * x)
    assert m == 1.0 and close(f.tolist(), want) and want[0] == 1.0
    f, m = mlxq.rotary_frequencies(128, 10000.0, "yarn", 16.0, 4096)
    at = lambda n: 128 * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
    lo, hi = math.floor(at(32)), math.ceil(at(1))
    want = []
    for i, x in enumerate(_freqs(128)):
        r = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        want.append(x / 16 * r + x * (1 - r))
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-15 and close(f.tolist(), want)
    assert 0 < lo < hi < 64


@pytest.mark.parametrize("kw", [dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=258), dict(base=1.0), dict(base=math.inf),
                                dict(scaling="none such"), dict(scaling="linear", factor=0.5), dict(scaling="ntk", rotary_dim=2, factor=2.0),
                                dict(scaling="yarn", factor=2.0), dict(scaling="llama3", factor=2.0, original_context=100, low=4.0, high=4.0)])
def test_frequencies_refusals(kw):
    with pytest.raises(mlxq.MlxqError):
        mlxq.rotary_frequencies(**{"rotary_dim": 64, **kw})


# ---- PagedCache: which sequence holds which page ----------------------------------------------------


class _Host(mlxq.PagedCache):
    """PagedCache over a list that stands for the pool: page -> the tokens last written there."""

    def __init__(self, pages, page_size=16):
        super().__init__(1, pages, 1, 16, page_size, torch.float32, "cpu")
        self.mem = [[] for _ in range(pages)]

    def _copy(self, src, dst, tables=None):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        for s, d in zip(src, dst):
            self.mem[d] = list(self.mem[s])


def _run(seed, steps=300):
    r = random.Random(seed)
    c, book = _Host(40), {}
    for step in range(steps):
        what = r.choice(["new", "batch", "batch", "fork", "free", "truncate", "compact"])
        live = sorted(book)
        try:
            if what == "new":
                book[c.new()] = []
            elif what == "batch" and live:
                seqs = r.sample(live, r.randint(1, min(4, len(live))))
                new = [r.randint(0, 20) for _ in seqs]
                before = {s: c.pages_of(s) for s in live}
                b = c.batch(seqs, new)
                assert b.q_starts.tolist() == [sum(new[:i]) for i in range(len(new) + 1)]
                assert b.max_q == max(new) and b.max_kv == max(c.length(s) for s in seqs)
                for row, s, n in zip(b.block_tables.tolist(), seqs, new):
                    pages = c.pages_of(s)
                    assert row[:len(pages)] == pages and set(row[len(pages):]) <= {-1} and pages[:len(before[s])] == before[s]
                    for i in range(n):
                        place = len(book[s])
                        page = pages[place // 16]
                        assert c._holders[page] == 1  # a page that is written is nobody else's
                        c.mem[page] = c.mem[page][:place % 16] + [(step, s, i)]
                        book[s].append((step, s, i))
                assert b.kv_lens.tolist() == [len(book[s]) for s in seqs]
            elif what == "fork" and live:
                seqs = [r.choice(live) for _ in range(r.randint(1, 3))]
                for s, n in zip(seqs, c.fork(seqs)):
                    book[n] = list(book[s])
            elif what == "free" and live:
                s = r.choice(live)
                c.free(s)
                del book[s]
            elif what == "truncate" and live:
                s = r.choice(live)
                n = r.randint(0, len(book[s]))
                c.truncate(s, n)
                book[s] = book[s][:n]
            elif what == "compact":
                used = c.compact()
                assert used == 40 - c.free_pages and all(p < used for s in book for p in c.pages_of(s))
        except mlxq.MlxqError as e:
            assert "free" in str(e)
        for s, tokens in book.items():
            pages = c.pages_of(s)
            assert c.length(s) == len(tokens) and len(pages) == -(-len(tokens) // 16)
            held = [t for i, p in enumerate(pages) for t in c.mem[p][:min(16, len(tokens) - 16 * i)]]
            assert held == tokens
        count = [0] * 40
        for s in book:
            for p in c.pages_of(s):
                count[p] += 1
        assert count == c._holders and sorted(c._free) == [p for p in range(40) if not count[p]]


@pytest.mark.parametrize("seed", range(8))
def test_paged_cache_book_keeping(seed):
    _run(seed)


def test_paged_cache_refusals():
    for kw in (dict(layers=0), dict(pages=0), dict(page_size=24), dict(page_size=8), dict(head_dim=72), dict(dtype=torch.float64)):
        with pytest.raises(mlxq.MlxqError):
            mlxq.PagedCache(**{**dict(layers=1, pages=4, heads=1, head_dim=16, device="cpu"), **kw})
    c = _Host(4)
    a = c.new()
    for call in (lambda: c.batch([a], [65]), lambda: c.batch([a, a], [1, 1]), lambda: c.batch([], []), lambda: c.batch([a], [-1]), lambda: c.batch([7], [1]),
                 lambda: c.fork([7]), lambda: c.free(7), lambda: c.length(7), lambda: c.truncate(a, 1)):
        with pytest.raises(mlxq.MlxqError):
            call()
    assert c.free_pages == 4 and c.length(a) == 0


def test_truncate_of_a_shared_page_in_a_full_pool():
    c = _Host(4)
    a = c.new()
    c.batch([a], [48])
    b, = c.fork([a])
    c.batch([b], [16])
    assert c.free_pages == 0
    with pytest.raises(mlxq.MlxqError):
        c.truncate(a, 40)  # its copy of the page would need a fifth
    assert c.length(a) == 48 and c.pages_of(a) == c.pages_of(b)[:3]
    c.truncate(b, 40)  # b's own fourth page holds the copy
    assert c.pages_of(b) == [0, 1, 3] and c.pages_of(a) == [0, 1, 2] and c._holders == [2, 2, 1, 1] and c.free_pages == 0


def test_layer_views():
    c = mlxq.PagedCache(3, 5, 2, 32, 32, torch.bfloat16, "cpu")
    for i in range(3):
        k, v = c.layer(i)
        assert (tuple(k.shape), tuple(v.shape)) == mlxq.cache_shapes(5, 2, 32, 32)
        assert k.data_ptr() == c.pool[i, 0].data_ptr() and v.data_ptr() == c.pool[i, 1].data_ptr()


def test_cpu_tensors_are_refused():
    c = mlxq.PagedCache(1, 5, 1, 16, 16, torch.float32, "cpu")
    s = c.new()
    x, b = torch.zeros(2, 1, 16), c.batch([s], [2])
    for call in (lambda: mlxq.cache_append(x, x, *c.layer(0), b), lambda: mlxq.paged_attention(x, *c.layer(0), b),
                 lambda: mlxq.rotary(x, torch.zeros(2, dtype=torch.int32), torch.zeros(4, 8, 2)),
                 lambda: mlxq.copy_pages(c.pool, torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="GPU tensors only"):
            call()
