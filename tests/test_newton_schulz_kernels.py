"""Every Newton-Schulz kernel in both orientations: values, and where NaN and infinity go."""
import math

import pytest
import torch

from tests.test_newton_schulz import BOUND, TYPES, exact, matrices, off
from tnn_b200.ops import _lib, raw

pytestmark = pytest.mark.gpu
# kernel (0: 128 x 64 tiles, 1: 128 x 128, 2: CTA pairs): shapes that take it, remainders on all sides among them
SHAPES = {
    0: [(3, 130, 140), (3, 140, 130), (1, 385, 1000), (1, 1000, 385)],
    1: [(9, 321, 1155), (9, 1155, 321), (20, 130, 700), (20, 700, 130), (40, 129, 257), (40, 257, 129)],
    2: [(80, 96, 200), (80, 200, 96), (60, 257, 300), (60, 300, 257)],
}
ALL = [(kernel, *shape) for kernel, shapes in SHAPES.items() for shape in shapes]


def _takes(kernel, count, m, n):
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the shapes are chosen for 148 SMs")
    assert _lib.load().tnnb_newton_schulz_kernel(count, m, n) == kernel


@pytest.mark.parametrize("kernel,count,m,n", ALL)
@pytest.mark.parametrize("kind", ["gauss", "gradient", "rank one"])
@pytest.mark.parametrize("dtype", TYPES)
def test_values(kernel, count, m, n, kind, dtype):
    _takes(kernel, count, m, n)
    g = matrices(count, m, n, kind, m + n)
    if dtype == torch.float16:
        g = g / g.flatten(1).norm(dim=1)[:, None, None] * math.sqrt(m * n)  # in its range
    g = g.to(dtype)
    got = raw.newton_schulz(g.cuda())
    assert off(got, exact(g)) < BOUND
    assert torch.equal(got, raw.newton_schulz(g.cuda()))


@pytest.mark.parametrize("kernel,count,m,n", ALL)
@pytest.mark.parametrize("steps", [1, 5])
def test_bad_numbers_fill_their_matrix_and_no_other(kernel, count, m, n, steps):
    _takes(kernel, count, m, n)
    g = matrices(count, m, n, "gauss").cuda()
    clean = raw.newton_schulz(g, steps)
    for bad in (math.nan, math.inf, -math.inf):
        for place in ((0, 0), (m - 1, n - 1), (m // 2, n // 3)):
            x = g.clone()
            x[(count // 2, *place)] = bad
            y = raw.newton_schulz(x, steps)
            assert bool(torch.isnan(y[count // 2]).all()), (bad, place)
            for i in (*range(count // 2), *range(count // 2 + 1, count)):
                assert torch.equal(y[i], clean[i]), (bad, place, i)
