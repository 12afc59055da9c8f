"""Registers of the microscaled, norm and routing kernels, read from the library's own code objects: none keeps values in scratch
memory, where one step of a product or one row of a norm would be written and read again."""
import re

from test_kernel_resources import kernels  # noqa: F401  (a fixture)


def test_no_spills(kernels):  # noqa: F811
    mine = {n: v for n, v in kernels.items() if re.search(r"\b(mx_\w+|rms_norm\w*|route\w*)_kernel", n)}
    assert len(mine) > 100
    assert not {n: v for n, v in mine.items() if v[1]}


def test_largest_tiles_leave_two_waves_a_simd(kernels):  # noqa: F811
    """The 256 x 256 tile: eight waves of at most 256 registers, accumulators included."""
    big = [v for n, v in kernels.items() if "mx_tile_kernel" in n and "256, 256" in n]
    assert len(big) == 2 and all(regs <= 256 for regs, _ in big)
