"""Orthogonalisation of matrices by Newton-Schulz products (csrc/kernels/newton_schulz.cu on CUDA, torch products on CPU)."""
from __future__ import annotations

import functools
import math
from typing import Sequence, Tuple

import torch

from . import _lib
from .gemm import LAUNCHES
from .vocab import _TYPES

#: ``a, b, c`` of the quintic ``a x + b x^3 + c x^5``: the largest slope at 0 of those that bring singular values into about [0.7, 1.2]
QUINTIC = (3.4445, -4.7750, 2.0315)
_DECLARED = False


def _library():
    global _DECLARED
    lib = _lib.load()
    if not _DECLARED:
        p, i, l, f = _lib.c_void_p, _lib.c_int, _lib.c_ll, _lib.c_float
        _lib.declare(lib, "tnnb_newton_schulz", [p, l, l, i, i, i, i, p, i, f, p, p, p, p, p, p, p, p, p, p])
        _DECLARED = True
    return lib


def _largest(poly: Sequence[float], upto: float) -> float:
    """Largest magnitude on ``[0, upto]`` of ``sum(poly[k] x^(first + 2 k))`` for the two polynomials below."""
    first, *coef = poly
    f = lambda x: abs(sum(c * x ** (first + 2 * k) for k, c in enumerate(coef)))
    # zeros of the derivative, a polynomial of degree one or two in x^2
    d = [c * (first + 2 * k) for k, c in enumerate(coef)]
    squares = []
    if len(d) == 2:
        squares = [-d[0] / d[1]] if d[1] else []
    elif d[2]:
        disc = d[1] * d[1] - 4 * d[0] * d[2]
        squares = [(-d[1] + s * math.sqrt(disc)) / (2 * d[2]) for s in (1, -1)] if disc >= 0 else []
    elif d[1]:
        squares = [-d[0] / d[1]]
    at = [math.sqrt(s) for s in squares if 0 < s < upto * upto]
    return max(f(x) for x in [upto] + at)


@functools.lru_cache(maxsize=64)
def _checked(coefficients: Tuple[float, ...]) -> object:
    """The coefficients as a C array, after a look at what they make of singular values in [0, 1]: the kernels keep X and X X^T
    times 2^12 and a + b A + c A A times 2^11 in fp16, whose largest number is 65504."""
    import ctypes

    upto = 1.0
    for k in range(0, len(coefficients), 3):
        a, b, c = coefficients[k:k + 3]
        if not all(math.isfinite(v) for v in (a, b, c)):
            raise ValueError(f"Newton-Schulz coefficients {(a, b, c)}")
        poly = _largest((2, b, c), upto)
        upto = 1.01 * _largest((1, a, b, c), upto)  # with room for what is rounded
        if abs(a) + poly > 30 or upto > 3.9:
            raise ValueError(f"Newton-Schulz coefficients {(a, b, c)} take singular values of [0, 1] to {upto:.3g} "
                             f"(factors of the products up to {abs(a) + poly:.3g}): at most 3.9 (30) are supported")
    return (ctypes.c_float * len(coefficients))(*coefficients)


def newton_schulz(g: torch.Tensor, steps: int = 5, coefficients: Sequence = QUINTIC, eps: float = 1e-7) -> torch.Tensor:
    """``steps`` Newton-Schulz steps on every matrix of ``g [..., m, n]``: ``X = G / (|G|_F + eps)``, then ``X <- a X + (b A + c A A) X``
    with ``A = X X^T`` (from the other side where ``m > n``). With the default ``coefficients`` five steps bring the singular values near
    one, which makes the result a stand-in for the orthogonal factor ``U V^T`` of ``G``. ``coefficients``: one triple for all
    steps or a triple for each.

    The result is bf16, packed, rounded once from fp32; the products take fp16 operands that are scaled into its range, X itself
    is carried with 22 bits up to the last two. A matrix of zeros stays one; NaN or infinity anywhere in a matrix make NaNs of it."""
    if g.dim() < 2 or not g.is_floating_point():
        raise ValueError(f"newton_schulz takes floating-point matrices, not {tuple(g.shape)} of {g.dtype}")
    steps = int(steps)
    flat = [float(v) for c in coefficients for v in (c if isinstance(c, (tuple, list)) else (c,))]
    if not 1 <= steps <= 64 or len(flat) not in (3, 3 * steps):
        raise ValueError(f"{len(flat)} coefficients for {steps} steps: one triple, or one per step, for 1 to 64 steps")
    flat = tuple(flat if len(flat) == 3 * steps else flat * steps)
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps {eps}")
    c_array = _checked(flat)
    m, n = g.shape[-2:]
    count = math.prod(g.shape[:-2])
    if m == 0 or n == 0 or count == 0:
        return torch.empty(g.shape, dtype=torch.bfloat16, device=g.device)
    if not g.is_cuda:
        x = g.float()
        norm = g.double().square().sum((-2, -1), keepdim=True).sqrt()
        x = (g.double() / (norm + eps)).float()
        for k in range(steps):
            a, b, c = flat[3 * k:3 * k + 3]
            gram = x @ x.mT if m <= n else x.mT @ x
            poly = b * gram + c * (gram @ gram)
            x = a * x + (poly @ x if m <= n else x @ poly)
        return x.to(torch.bfloat16)
    code = _TYPES.get(g.dtype)
    if code is None:
        raise TypeError(f"newton_schulz on {g.dtype}; the kernels take bfloat16, float16 and float32")
    if max(m, n) >= 1 << 24:
        raise ValueError(f"matrices of {m} x {n}")
    with _lib.device_of(g):
        x = g.reshape(count, m, n)
        if (x.stride(2) != 1 and n > 1) or (m > 1 and x.stride(1) < n):
            x = x.contiguous()
        out = torch.empty(g.shape, dtype=torch.bfloat16, device=g.device)
        item, ld = x.stride(0), x.stride(1) if m > 1 else n
        low = min(m, n)
        size_x, size_s = 2 * m * ((n + 7) // 8 * 8), 2 * low * ((low + 7) // 8 * 8)  # bytes per matrix
        most = 4096  # matrices per call
        for i in range(0, count, most):
            k = min(most, count - i)
            parts = [(k * s + 255) // 256 * 256 for s in (size_x, size_x, size_x, size_s, size_s, 512, 12 * steps + 4)]
            work = torch.empty(sum(parts), dtype=torch.uint8, device=g.device)
            at = [work.data_ptr() + sum(parts[:j]) for j in range(7)]
            rc = _library().tnnb_newton_schulz(x.data_ptr() + i * item * x.element_size(), item, ld, code, k, m, n, _address(c_array), steps,
                                               float(eps), out.data_ptr() + i * m * n * 2, *at, _lib.status_addr(g.device),
                                               _lib.raw_stream())
            _lib.check_rc(rc, "newton_schulz")
            LAUNCHES["count"] += 3
    return out


def _address(array) -> int:
    import ctypes

    return ctypes.addressof(array)
