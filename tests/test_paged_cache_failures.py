"""PagedCache when a call fails on the device (no memory for the step's tables or the list of pages to copy): the book is what it was,
so that the call can be made again.  On the CPU."""
import copy

import pytest
import torch

import mlxq


class _Failing(mlxq.PagedCache):
    """A PagedCache whose device fails while `broken`; copies are listed."""

    def __init__(self, pages):
        super().__init__(1, pages, 1, 16, 16, torch.float32, "cpu")
        self.broken, self.copies = False, []
        self.pool = self

    @property
    def device(self):  # of the pool: where the step's tables go
        if self.broken:
            raise torch.cuda.OutOfMemoryError("out of memory")
        return torch.device("cpu")

    def _copy(self, src, dst, tables=None):
        self.device
        self.copies.append((list(src), list(dst)))

    def book(self):
        return copy.deepcopy((sorted(self._free), self._holders, self._seqs, self.free_pages))


def _cache():
    c = _Failing(8)
    a, b = c.new(), c.new()
    c.batch([a, b], [40, 10])
    d, = c.fork([a])
    return c, a, b, d


@pytest.mark.parametrize("call", [lambda c, a, b, d: c.batch([a, b], [30, 3]), lambda c, a, b, d: c.fork([a, b]), lambda c, a, b, d: c.truncate(d, 20),
                                  lambda c, a, b, d: c.truncate(a, 5)],
                         ids=["batch", "fork", "truncate", "truncate more"])
def test_a_failed_call_changes_nothing(call):
    c, a, b, d = _cache()
    want, _ = _cache()[0], None
    before = c.book()
    c.broken = True
    with pytest.raises(torch.cuda.OutOfMemoryError):
        call(c, a, b, d)
    assert c.book() == before
    c.broken = False
    first, second = call(c, a, b, d), call(want, a, b, d)
    assert c.book() == want.book()
    if isinstance(first, mlxq.CacheBatch):
        assert torch.equal(first.kv_lens, second.kv_lens) and torch.equal(first.block_tables, second.block_tables)


def test_a_failed_compaction_changes_nothing():
    c, a, b, d = _cache()
    c.free(b)
    c.truncate(a, 0)
    before = c.book()
    c.broken = True
    with pytest.raises(torch.cuda.OutOfMemoryError):
        c.compact()
    assert c.book() == before
    c.broken = False
    assert c.compact() == 3
