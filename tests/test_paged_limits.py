"""Sizes past what the paged-cache kernels count in 31 bits are refused before anything is launched, and what the launches are
planned for is bounded.  On the CPU: the checks and the plan need no device."""
import ctypes

import pytest

from mlxq import _lib

P = 4096  # any aligned address: nothing below gets as far as reading it


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _attention(lib, T, Hq, Hkv, D=64, dtype=1, B=3, max_q=1, max_kv=64, width=4, size=False, **opts):
    """(status, message) of a call whose workspace is too small, or its workspace size."""
    cache = _lib.PagedCacheView(P, P, Hkv * 16 * D, Hkv * 16 * D, 2 ** 30, 16, Hkv, D, dtype)
    batch = _lib.PagedBatch(P, P, P, B, width, width, max_q, max_kv)
    o = _lib.Attention(**{**dict(scale=0.125, causal=1, window=0, softcap=0.0, prefix_lens=None, alibi_slopes=None, sinks=None), **opts})
    q = _lib.Heads(P, Hq, Hq * D, D)
    r = ctypes.byref
    if size:
        return lib.mlxq_paged_attention_workspace_size(T, Hq, r(cache), r(batch), r(o))
    rc = lib.mlxq_paged_attention(r(q), T, r(cache), r(batch), r(o), r(q), None, 0, None)
    return rc, lib.mlxq_last_error().decode()


LONG = dict(B=1, max_kv=10 ** 6, width=10 ** 5)


@pytest.mark.parametrize("T,Hq,Hkv", [(2 ** 26, 64, 2), (2 ** 30 - 1, 2, 1), (2 ** 30 - 1, 65535, 1), (2 ** 16, 32768, 1)])
def test_rows_past_31_bits_are_refused(lib, T, Hq, Hkv):
    """A key head's rows, (token, query head) pairs, and a tile after them are counted in 31 bits."""
    for D, dtype, max_q in ((64, 1, 1), (64, 1, T), (256, _lib.MLXQ_FLOAT16, 500), (64, 0, T)):
        kw = dict(D=D, dtype=dtype, max_q=max_q, **LONG)
        rc, msg = _attention(lib, T, Hq, Hkv, **kw)
        assert rc == _lib.MLXQ_EINVAL and "rows" in msg, msg
        assert _attention(lib, T, Hq, Hkv, size=True, **kw) == 0


@pytest.mark.parametrize("T,Hq,Hkv", [(2 ** 25, 64, 64), (2 ** 30 - 1, 32, 32)])
def test_results_past_31_bits_are_not_split(lib, T, Hq, Hkv):
    """Where sequences are split, a row of results of every query head has a place in the workspace, counted in 31 bits."""
    assert _attention(lib, T, Hq, Hkv, size=True, **LONG) == 0


@pytest.mark.parametrize("window", [10 ** 6, 2 ** 40, 2 ** 62, 2 ** 63 - 1])
def test_a_window_past_every_context_plans_as_none(lib, window):
    """"No limit" is often written as the largest integer."""
    for kw in (dict(T=2, Hq=8, Hkv=2, B=2, max_kv=150001, width=10 ** 4), dict(T=300, Hq=8, Hkv=2, B=1, max_q=300, max_kv=9000, width=10 ** 3)):
        want = _attention(lib, size=True, **kw)
        assert want > 0 and _attention(lib, size=True, window=window, **kw) == want


def _splits(lib, Hq=4, Hkv=2, D=64, **kw):
    """Splits of a plan, from its workspace: rows of S x D sums, of S (maximum, sum) pairs and of counts, each rounded up."""
    T = kw["T"]
    need = _attention(lib, Hq=Hq, Hkv=Hkv, D=D, size=True, **kw)
    up = lambda b: -(-b // 256) * 256  # noqa: E731
    return next((S for S in range(2, 300) if up(T * Hq * S * D * 4) + up(T * Hq * S * 8) + up(T * Hq * 4) == need), 1 if need == 0 else None)


@pytest.mark.parametrize("T,max_kv", [(500, 16384), (16384, 16384), (40, 9000)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_rows_that_see_past_their_window_are_planned_for(lib, T, max_kv, dtype):
    """With a window, a causal row sees no more tokens than that; one that sees all later tokens, up to as many more as the step
    has, and no split may be left with most of them.  Prefixes, which are on the device, change no plan."""
    kw = dict(T=T, B=1, max_q=T, max_kv=max_kv, width=10 ** 4, dtype=dtype, window=128)
    reach = min(max_kv, 128 + T)
    plain = _splits(lib, **{**kw, "max_kv": reach, "window": 0})  # the same rows over as many tokens, all of them seen
    assert _splits(lib, causal=0, **kw) == plain
    assert _splits(lib, prefix_lens=P, **kw) == _splits(lib, **kw) <= max(plain, 2)


@pytest.mark.parametrize("hint", [2 ** 31, 2 ** 47, 2 ** 62, 2 ** 63 - 1])
def test_hints_past_every_step_plan_alike(lib, hint):
    """max_q and max_kv are hints of any size: neither is multiplied past 63 bits."""
    kw = dict(T=300, Hq=8, Hkv=2, B=2, width=10 ** 3, dtype=0)
    want = _attention(lib, size=True, **kw, max_q=2 ** 30, max_kv=2 ** 30)
    assert want > 0 and _attention(lib, size=True, **kw, max_q=hint, max_kv=2 ** 30) == want
    assert _attention(lib, size=True, **kw, max_q=hint, max_kv=hint) == want
    assert _attention(lib, size=True, **{**kw, "dtype": 1}, max_q=hint, max_kv=hint) == \
        _attention(lib, size=True, **{**kw, "dtype": 1}, max_q=2 ** 30, max_kv=2 ** 30)


@pytest.mark.parametrize("B,new,Hq,Hkv,D,max_kv", [(256, 1, 64, 8, 128, 131072), (256, 2, 64, 8, 128, 131072), (2048, 1, 8, 1, 64, 32768),
                                                   (100, 2, 32, 8, 256, 10 ** 6), (4096, 4, 32, 8, 128, 10 ** 6), (300, 1, 32, 1, 64, 2 ** 24)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_many_sequences_under_a_long_hint(lib, B, new, Hq, Hkv, D, max_kv, dtype):
    """A replayed step is planned for the longest context; how many sequences it has bounds the splits, and with them the workspace
    and the workgroups that find nothing to do."""
    kw = dict(T=B * new, B=B, max_q=new, max_kv=max_kv, width=max_kv // 16, dtype=dtype)
    S = _splits(lib, Hq=Hq, Hkv=Hkv, D=D, **kw)
    assert S is not None and S * B * Hkv <= 16 * 3 * 256 + B * Hkv
    assert _attention(lib, Hq=Hq, Hkv=Hkv, D=D, size=True, **kw) <= 2 ** 28 + 2 ** 24


def test_the_longest_tables_and_the_most_sequences(lib):
    kw = dict(T=2 ** 24 - 1, Hq=64, Hkv=64, B=2 ** 24 - 1, width=2 ** 31 - 1)
    assert _attention(lib, size=True, max_kv=2 ** 63 - 1, **kw) == _attention(lib, size=True, max_kv=2 ** 30 - 1, **kw) == 0


def test_more_tokens_than_hinted(lib):
    """max_q is a hint: the workspace stays bounded for a step that has many more tokens."""
    assert _attention(lib, T=100000, Hq=32, Hkv=8, D=128, B=1, max_q=1, max_kv=131072, width=8192, size=True) <= 2 ** 28 + 2 ** 24


def test_few_sequences_are_still_split(lib):
    """768 tokens a split where the chip has room for the workgroups."""
    assert _splits(lib, Hq=64, Hkv=8, T=48, B=48, max_kv=6000, width=375) == 8
    assert _splits(lib, Hq=28, Hkv=4, D=128, T=2, B=2, max_kv=150001, width=9376) == 196
    assert _splits(lib, Hq=32, Hkv=8, D=128, T=8, B=1, max_q=8, max_kv=131072, width=8192) > 40
