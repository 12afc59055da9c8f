"""paged_attention with caps from far below the scores to far above them, in every type: cap tanh(z / cap) is a step for the first
and z itself for the last.  Bounds: paged_ref, whose error of a score, 16 2^-24 (1 + |z|), knows no cap; the cap's own
arithmetic has to stay within it."""
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


def _check(mlxq, pr, opts):
    given = {{"slopes": "alibi_slopes"}.get(n, n): v.cuda() if isinstance(v, torch.Tensor) else v for n, v in opts.items()}
    got = mlxq.paged_attention(pr.q.cuda(), *pr.cache(), pr.batch(), **given)
    want, tol = ref.attention(pr, **opts)
    d = (got.double().cpu() - want).abs()
    print(f"    error / bound {float((d / (tol + 1e-30)).max()):.3f}", flush=True)
    assert torch.isfinite(got).all() and (d <= tol).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("cap", [1e-30, 1e-3, 0.5, 4.0, 30.0, 300.0, 1e4, 1e5, 1e6, 1e7, 1e9, 1e15, 1e30, 3.4e38])
@pytest.mark.parametrize("lens", [[(1, 70), (3, 40)], [(70, 130), (1, 90)]], ids=["step", "chunk"])
def test_caps_of_any_size(mlxq, dtype, cap, lens):
    banner("paged_attention cap", dtype, cap, lens)
    _check(mlxq, ref.Problem(7, lens, 1, 2, 64, 16, dtype), dict(softcap=cap))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("std", [0.05, 1.5, 4.0])
@pytest.mark.parametrize("cap", [1e4, 1e6])
def test_caps_above_small_and_large_scores(mlxq, dtype, std, cap):
    banner("paged_attention cap, scores", dtype, std, cap)
    opts = dict(softcap=cap, slopes=torch.tensor([0.25, 0.0]))
    _check(mlxq, ref.Problem(11, [(40, 150), (1, 60)], 1, 2, 128, 32, dtype, std), opts)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_cap_out_of_reach_changes_nothing_that_bf16_shows(mlxq, D):
    """A cap of 1e9 differs from none by the scores' last bits: both are within the bound of the result without one."""
    pr = ref.Problem(3, [(1, 30), (60, 90)], 2, 1, D, 16, BF16)
    q, (k, v), b = pr.q.cuda(), pr.cache(), pr.batch()
    a, c = mlxq.paged_attention(q, k, v, b), mlxq.paged_attention(q, k, v, b, softcap=1e9)
    _, tol = ref.attention(pr)
    assert ((a.double() - c.double()).abs().cpu() <= 2 * tol).all()
