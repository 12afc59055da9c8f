"""examples/paged_decode.py end to end."""
import importlib.util
import os

import pytest

from gpu_util import banner

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decode.py")


@pytest.mark.parametrize("bits", [4, 8])
def test_serving_matches_a_pass_without_a_cache(bits):
    """Both paths round the same ten bf16 intermediates a block (2^-9 / sqrt 3 each) and differ in the attention's
    and the projections' order of sums: two blocks give about sqrt(2 * 20) * 1.1e-3 = 7e-3, allowed three times that.
    A wrong or missing token changes the logits by tens of percent."""
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    banner("example", bits)
    lines = []
    worst = m.run(layers=2, hidden=512, steps=5, bits=bits, prompts=(70, 17, 33, 1), say=lines.append)
    print("\n".join(lines), flush=True)
    assert worst <= 2.1e-2
    assert len([s for s in lines if s.startswith("sequence")]) == 4
