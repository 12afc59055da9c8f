"""A cache whose pages share memory is refused on every path: the kernels step from page to page by at least a page, so
the last pages of such a view would lie past its memory."""
import pytest
import torch

import mlxq


def _shared(device, pages=9):
    """One page of memory shown as many, and the rest of a step."""
    ks, vs = mlxq.cache_shapes(1, 2, 16, 64)
    k, v = (torch.zeros(s, dtype=torch.bfloat16, device=device) for s in (ks, vs))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    batch = mlxq.CacheBatch(i32([[0]]), i32([0, 1]), i32([1]), 1, 1)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=device)
    return x, k, v, k.expand(pages, *ks[1:]), v.expand(pages, *vs[1:]), batch


def _refused(device):
    x, k, v, kk, vv, batch = _shared(device)
    apart_k, apart_v = (torch.zeros(9, *t.shape[1:], dtype=t.dtype, device=device) for t in (k, v))
    half = torch.zeros(9 * 2048, dtype=torch.bfloat16, device=device).as_strided(apart_k.shape, (1024, *apart_k.stride()[1:]))
    for what, a, b in (("k_cache", kk, vv), ("k_cache", kk, apart_v), ("v_cache", apart_k, vv), ("k_cache", half, apart_v)):
        for call in (lambda: mlxq.paged_attention(x, a, b, batch), lambda: mlxq.paged_attention(x, a, b, batch, out=torch.empty_like(x)),
                     lambda: mlxq.cache_append(x, x, a, b, batch)):
            with pytest.raises(mlxq.MlxqError, match=f"pages of {what} overlap") as e:
                call()
            assert e.value.status == 1


def test_shared_pages_are_refused():
    _refused("cpu")


@pytest.mark.gpu
def test_shared_pages_are_refused_on_the_gpu():
    _refused("cuda")


@pytest.mark.gpu
def test_one_page_of_any_stride():
    """A single page has no next one: its stride means nothing."""
    x, k, v, _, _, batch = _shared("cuda")
    x += 1
    one = [t.as_strided(t.shape, (0, *t.stride()[1:])) for t in (k, v)]
    mlxq.cache_append(x, x, *one, batch)
    assert torch.equal(mlxq.paged_attention(x, *one, batch), x)
