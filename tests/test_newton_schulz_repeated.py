"""Newton-Schulz products of matrices in which few numbers repeat (diagonal ones, permutations, constants): equal numbers are rounded
alike, so that the fp16 roundings of the products do not average out as they do among many different elements."""
import math

import pytest
import torch

from tests.test_newton_schulz import TYPES, exact, off
from tnn_b200.ops import raw
from tnn_b200.ops.orthogonal import QUINTIC

HALF = 2.0 ** -11  # largest relative error of a rounding to fp16
WORST = 0.0271     # of one singular value, as documented: the largest of the scan below


def _quintic(x):
    a, b, c = QUINTIC
    return a * x + b * x ** 3 + c * x ** 5


def _chain(x, steps=5):
    """What becomes of one singular value: the roundings of csrc/kernels/newton_schulz.cu, one element per row and column."""
    a, b, c = QUINTIC

    def half(v):
        return v.float().half().double()

    X = x * 4096.0
    hi = half(X)
    lo = half(X - hi)
    for k in range(steps):
        A = half(hi * hi / 4096.0)
        folded = k + 2 >= steps
        B = half(((a if folded else 0.0) + b * A / 4096.0 + c * (A / 4096.0) ** 2) * 2048.0)
        X = (0.0 if folded else a * (hi + lo)) + B * hi / 2048.0
        hi = half(X)
        lo = half(X - hi)
    return (X / 4096.0).float().bfloat16().double()


def _bound(x, steps=5):
    """Relative error of a singular value ``x`` if all roundings err alike: in a step the operand of both products (three times half a step
    in A and A^2, with A's own), B and the operand beside it; in front of the last two steps and in B's diagonal X's own; what was off
    before is multiplied by the quintic's slope. (A twentieth more for products of errors.)"""
    a, b, c = QUINTIC
    d = x * 2.0 ** -22
    for k in range(steps):
        folded = k + 2 >= steps
        B = b * x * x + c * x ** 4
        new = x * HALF * (3 * abs(b * x * x + 2 * c * x ** 4) + 2 * abs(B + a if folded else B))
        y = _quintic(x)
        d = abs(a + 3 * b * x * x + 5 * c * x ** 4) * d + new + abs(y) * (2.0 ** -8 if k + 1 == steps else HALF if k + 3 >= steps else 2.0 ** -22)
        x = y
    return 1.05 * d / abs(x)


def test_worst_singular_value():
    x = torch.exp(torch.linspace(math.log(1e-4), 0, 400001, dtype=torch.float64))
    ref = x
    for _ in range(5):
        ref = _quintic(ref)
    error = (_chain(x) - ref).abs() / ref.abs()
    assert 0.026 < float(error.max()) < WORST
    assert all(float(error[i]) <= _bound(float(x[i])) for i in range(0, 400001, 1000))


def _matrix(kind):
    gen = torch.Generator().manual_seed(3)
    name, *size = kind.split()
    m, n = int(size[0]), int(size[-1])
    g = torch.zeros(m, n)
    if name == "constant":
        return g + 0.37
    if name == "diagonal":
        g[range(m), range(m)] = torch.exp(-6 * torch.rand(m, generator=gen))
    elif name == "permutation":
        g[torch.randperm(m, generator=gen), torch.arange(m)] = torch.randint(0, 2, (m,), generator=gen) * 2.0 - 1.0
    else:
        g[range(m), range(m)] = 1.0
        if name == "noisy":
            g += torch.randn(m, n, generator=gen) * 1e-3
    return g


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["identity 1", "identity 2", "identity 43", "identity 343", "identity 382", "identity 382 764", "identity 1024",
                                  "permutation 382", "permutation 97 200", "diagonal 2", "diagonal 50", "diagonal 300 700", "constant 256 768",
                                  "constant 5 3", "constant 700 130", "noisy 382", "noisy 382 500"])
@pytest.mark.parametrize("count", [1, 30])
def test_repeated_numbers(kind, count):
    g = _matrix(kind)
    sigma = torch.linalg.svdvals(g.double() / g.double().norm())
    bound = max(_bound(float(s)) for s in sigma[sigma > 1e-6])
    ref = exact(g[None])
    for x in (g, g.mT):
        for dtype in TYPES[:1] if "noisy" in kind or "diagonal" in kind else TYPES:
            if kind.startswith("constant"):
                x = x.to(dtype).float()
            got = raw.newton_schulz(x.to(dtype).cuda().expand(count, *x.shape))
            error = off(got, (ref if x.shape == g.shape and torch.equal(x, g) else exact(x[None])).expand(count, *x.shape))
            assert error < bound, (kind, dtype, error, bound)
            if kind.split()[0] != "constant" and "noisy" not in kind:
                assert error < WORST  # one element per row and column: the chain itself
