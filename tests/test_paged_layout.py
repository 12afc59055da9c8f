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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("head_dim,page", [(32, 16), (64, 64), (128, 16), (256, 128)])
def test_the_pages_dimension(monkeypatch, dtype, head_dim, page):
    """By default the pages are the dimension before a pool's own, for stacks of key pools and of value pools alike."""
    seen = []

    class Fast:
        @staticmethod
        def copy_pages(cache, src, dst, tables, dim):
            seen.append(dim)
            return True

    monkeypatch.setattr(mlxq._lib, "_fast", Fast)
    for shape in mlxq.cache_shapes(3, 2, page, head_dim, dtype):
        for lead in ((), (4,), (4, 2)):
            mlxq.copy_pages(torch.empty(*lead, *shape, dtype=dtype), None, None)
            assert seen.pop() == len(lead), (lead, shape)
            mlxq.copy_pages(torch.empty(*lead, *shape, dtype=dtype), None, None, dim=7)
            assert seen.pop() == 7


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(), (3,)])
def test_copies_in_a_stack_of_value_pools(lead):
    v = torch.arange(24, device="cuda", dtype=torch.float32).view(*lead, -1, 1, 1, 1, 1) if lead else torch.arange(24., device="cuda").view(-1, 1, 1, 1, 1)
    v = v.expand(*v.shape[:len(lead) + 1], 2, 4, 64, 4).contiguous()
    want = v.clone()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    mlxq.copy_pages(v, i32(0, 5), i32(2, 1))
    at = (slice(None),) * len(lead)
    want[(*at, 2)], want[(*at, 1)] = want[(*at, 0)].clone(), want[(*at, 5)].clone()
    assert torch.equal(v, want)
