"""Newton-Schulz orthogonalisation: CPU form and kernels against the definition in 64 bits."""
import math

import pytest
import torch

from tnn_b200.ops import raw
from tnn_b200.ops.orthogonal import QUINTIC, _checked

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def exact(g, steps=5, coefficients=QUINTIC, eps=1e-7):
    x = g.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for k in range(steps):
        a, b, c = coefficients if isinstance(coefficients[0], float) else coefficients[k]
        left = x.shape[-2] <= x.shape[-1]
        gram = x @ x.mT if left else x.mT @ x
        poly = b * gram + c * gram @ gram
        x = a * x + (poly @ x if left else x @ poly)
    return x


def matrices(count, m, n, kind, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g)

    if kind == "gauss":
        return normal(count, m, n)
    if kind == "gradient":  # products of few tokens' signals of uneven strength
        out = normal(count, 32, m) * torch.exp(normal(count, 1, m))
        inp = normal(count, 32, n) * torch.exp(0.5 * normal(count, 1, n)) + normal(count, 1, n)
        return (out.mT @ inp) * 1e-5 + 1e-7 * normal(count, m, n)
    return normal(count, m, 1) @ normal(count, 1, n) + 0.003 * normal(count, m, n)  # rank one and noise


def off(got, ref):
    """Relative error in the 2-norm of each matrix, the worst of them."""
    d = (got.double().cpu() - ref).flatten(-2).norm(dim=-1) / ref.flatten(-2).norm(dim=-1).clamp_min(1e-300)
    return float(d.max())


# Rounding to bf16: half a step, 2^-9 to 2^-8 of a value, root mean square at most 2^-8 / sqrt(3) = 0.0023 (2-norm of the matrix).
ROUNDED = 2.0 ** -8 / math.sqrt(3)
# fp16 operands: a product's operands are off by at most 2^-11 each, root mean square 2^-11 / sqrt(3) = 0.00028. In a step three roundings
# reach X (of X in A and in B X, of A, of B), each times coefficients of size |b| sigma^2 + 2 |c| sigma^4 < 8 at most; errors of
# earlier steps are multiplied by the quintic's slope, which is above one while the matrix grows by the same factor (and near singular
# values of 1.2, up to 3.9, which few of a matrix's are: not so where a matrix has only a few), so that five steps
# add up to at most sqrt(5 * 4) * 8 / 2 (the mean of sigma^2 over the steps is below 1/2) times that.
OPERANDS = 2.0 ** -11 / math.sqrt(3) * math.sqrt(20) * 4
BOUND = ROUNDED + OPERANDS


@pytest.mark.parametrize("m,n", [(1, 1), (3, 7), (40, 24), (64, 64)])
@pytest.mark.parametrize("kind", ["gauss", "gradient", "rank one"])
def test_cpu_form(m, n, kind):
    g = matrices(2, m, n, kind)
    assert off(raw.newton_schulz(g), exact(g)) < ROUNDED + 1e-4
    assert raw.newton_schulz(g[0]).shape == (m, n) and raw.newton_schulz(g[0]).dtype == torch.bfloat16


def test_singular_values_end_near_one():
    g = matrices(1, 48, 80, "gauss")[0]
    s = torch.linalg.svdvals(raw.newton_schulz(g).float())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


def test_zeros_and_bad_numbers():
    g = torch.zeros(3, 8, 12)
    g[1, 2, 3], g[2] = math.nan, 1.0
    y = raw.newton_schulz(g)
    assert torch.equal(y[0], torch.zeros(8, 12, dtype=torch.bfloat16)) and bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[2]).all())


def test_refusals():
    g = torch.zeros(4, 6)
    for error, call in [
        (ValueError, lambda: raw.newton_schulz(g[0])),
        (ValueError, lambda: raw.newton_schulz(g.long())),
        (ValueError, lambda: raw.newton_schulz(g, steps=0)),
        (ValueError, lambda: raw.newton_schulz(g, steps=65)),
        (ValueError, lambda: raw.newton_schulz(g, coefficients=(1.0, 2.0))),
        (ValueError, lambda: raw.newton_schulz(g, steps=3, coefficients=[QUINTIC] * 2)),
        (ValueError, lambda: raw.newton_schulz(g, coefficients=(30.0, -4.0, 2.0))),  # singular values leave fp16's range
        (ValueError, lambda: raw.newton_schulz(g, coefficients=(math.nan, 0.0, 0.0))),
        (ValueError, lambda: raw.newton_schulz(g, eps=-1.0)),
    ]:
        with pytest.raises(error):
            call()
    assert raw.newton_schulz(torch.zeros(0, 4, 6)).shape == (0, 4, 6)
    _checked(QUINTIC * 5)
    _checked((1.5, -0.5, 0.0) * 7)  # the cubic


# extents around the tiles' (128 and 256), around whole vectors, single rows and columns; batches that take either kernel
SHAPES = [(1, 1, 1), (2, 1, 40), (2, 40, 1), (1, 5, 7), (3, 64, 64), (1, 127, 129), (2, 130, 257), (2, 300, 65), (1, 256, 512), (1, 520, 264),
          (40, 300, 310), (30, 520, 257), (80, 96, 200)]


@gpu
@pytest.mark.parametrize("count,m,n", SHAPES)
@pytest.mark.parametrize("kind", ["gauss", "gradient", "rank one"])
@pytest.mark.parametrize("dtype", TYPES)
def test_kernels(count, m, n, kind, dtype):
    g = matrices(count, m, n, kind, m + n)
    if dtype == torch.float16:
        g = g / g.flatten(1).norm(dim=1)[:, None, None] * math.sqrt(m * n)  # in its range
    g = g.to(dtype)
    got = raw.newton_schulz(g.cuda())
    assert got.shape == g.shape and got.dtype == torch.bfloat16 and off(got, exact(g)) < BOUND
    assert torch.equal(got, raw.newton_schulz(g.cuda()))


@gpu
@pytest.mark.parametrize("steps,coefficients", [(1, QUINTIC), (2, QUINTIC), (3, [(3.4445, -4.775, 2.0315), (2.5, -2.5, 0.9), (1.5, -0.5, 0.0)])])
def test_other_steps(steps, coefficients):
    for m, n in ((70, 200), (200, 70)):
        g = matrices(2, m, n, "gauss")
        assert off(raw.newton_schulz(g.cuda(), steps, coefficients), exact(g, steps, coefficients)) < BOUND


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_any_magnitude(scale):
    g = matrices(2, 60, 90, "gauss") * scale
    ref = exact(g)
    got = raw.newton_schulz(g.cuda())
    if scale == 1e-30:  # far below eps: nothing is left in bf16's comparison, the norm must not overflow or vanish
        assert float(got.float().abs().max()) < 1e-10
    else:
        assert off(got, ref) < BOUND


@gpu
def test_strided_batches():
    wide = torch.randn(3, 80, 150)
    for cut in (wide[:, :, :96], wide[:, 3:67, 5:140], wide[::2], wide.mT, wide[1], wide[:, :1], wide[:1].expand(3, 80, 150)):
        dev = wide.cuda().as_strided(cut.shape, cut.stride(), cut.storage_offset())
        assert off(raw.newton_schulz(dev), exact(cut)) < BOUND


@gpu
def test_zeros_and_bad_numbers_on_the_gpu():
    g = torch.zeros(3, 130, 140)
    g[1, 2, 3], g[2] = math.nan, 1.0
    y = raw.newton_schulz(g.cuda()).cpu()
    assert torch.equal(y[0], torch.zeros(130, 140, dtype=torch.bfloat16)) and bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[2]).all())
    g[1, 2, 3] = math.inf
    y = raw.newton_schulz(g.cuda()).cpu()
    assert bool(torch.isnan(y[1]).any()) and bool(torch.isfinite(y[2]).all())
    with pytest.raises(TypeError):
        raw.newton_schulz(torch.zeros(4, 4, dtype=torch.float64, device="cuda"))


@gpu
def test_captured_and_replayed():
    g = matrices(3, 150, 200, "gradient").cuda()
    raw.newton_schulz(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = raw.newton_schulz(g)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (5, 6):
        g.copy_(matrices(3, 150, 200, "gauss", seed))
        graph.replay()
        assert torch.equal(out, raw.newton_schulz(g))


@gpu
def test_two_streams_at_once():
    """Two calls in flight on two streams: each kernel's blocks run together or not yet, and neither sees the other's matrices."""
    g = [matrices(3, 150, 200, "gradient", s).cuda() for s in (1, 2)]
    alone = [raw.newton_schulz(x) for x in g]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(raw.newton_schulz(g[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, alone[i]) for x in got[i])


@gpu
def test_offsets_beyond_32_bits():
    far = 2 ** 31 + 16  # elements between two matrices, and between two rows of one
    space = torch.empty(far + 4096, dtype=torch.bfloat16, device="cuda")
    for shape, strides in (((2, 20, 30), (far, 30, 1)), ((2, 30), (far, 1))):
        g = space.as_strided(shape, strides)
        g.copy_(torch.randn(shape))
        assert torch.equal(raw.newton_schulz(g), raw.newton_schulz(g.contiguous()))
