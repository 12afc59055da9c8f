"""paged_attention looks up no page that lies before every row's window: entries there may name nothing, and the results are those
of the window alone, in steps, chunks and split sequences of every type."""
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


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("entry", [-1, 2 ** 31 - 1, 10 ** 6])
@pytest.mark.parametrize("new,length,window,D", [(1, 150, 40, 64), (6, 150, 40, 64), (60, 150, 40, 64), (60, 400, 33, 128), (130, 500, 129, 256),
                                                 (3, 3000, 900, 64), (70, 3000, 1000, 128)])
def test_entries_before_the_window_are_not_looked_up(mlxq, dtype, entry, new, length, window, D):
    banner("paged_attention window", dtype, entry, new, length, window, D)
    pr = ref.Problem(new, [(new, length), (2, 70)], 1, 2, D, 16, dtype)
    b = pr.batch()
    first = length - new + 1 - window  # the first token that any row sees
    assert first >= 16
    b.block_tables[0, :first // 16] = entry
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), b, window=window)
    want, tol = ref.attention(pr, window=window)
    assert torch.isfinite(got).all() and ((got.double().cpu() - want).abs() <= tol).all()
    # one page more, and the rows that see it are NaN, the others unchanged
    b.block_tables[0, first // 16] = entry
    bad = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), b, window=window)
    place = torch.arange(length - new, length)
    sees = torch.zeros(pr.T, dtype=torch.bool)
    sees[:new] = place + 1 - window < (first // 16 + 1) * 16
    assert bad.cpu()[sees].isnan().all() and torch.equal(bad.cpu()[~sees], got.cpu()[~sees])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_window_of_the_largest_integer_hides_nothing(mlxq, dtype):
    banner("paged_attention window 2^63 - 1", dtype)
    pr = ref.Problem(5, [(1, 2000), (50, 90)], 1, 2, 64, 16, dtype)
    q, (k, v), b = pr.q.cuda(), pr.cache(), pr.batch()
    assert torch.equal(mlxq.paged_attention(q, k, v, b, window=2 ** 63 - 1), mlxq.paged_attention(q, k, v, b))
