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
def test_split_results_past_31_bits_are_refused(lib, T, Hq, Hkv):
    """Where sequences are split, a row of results of every query head has a place in the workspace, counted in 31 bits: refused
    before the first kernel, not between it and the join."""
    rc, msg = _attention(lib, T, Hq, Hkv, **LONG)
    assert rc == _lib.MLXQ_EINVAL and "too large" in msg, msg
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
