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

    The result is bf16, packed, rounded once from fp32. On CUDA the products take fp16 operands that are scaled into its range, X itself
    is carried with 22 bits up to the last two. Matrices of many different elements come out 0.2 % of the 2-norm off, of which most
    is the result's rounding. Where few numbers repeat (diagonal matrices, permutations, constants, a few elements at all) their
    roundings do not average out: with the default coefficients identities are up to 1.2 % off, any one singular value above 1e-4 of the
    norm 2.7 % at most. On CPU the products are fp32. A matrix of zeros stays one; NaN or infinity anywhere in a matrix make NaNs of it.
    There is no derivative on CUDA (on CPU torch records its products)."""
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


# ------------------------------------------------------------------------- the optimizer's element-wise passes
_MUON_DECLARED = False


def _muon_library():
    global _MUON_DECLARED
    lib = _lib.load()
    if not _MUON_DECLARED:
        p, i, l, f = _lib.c_void_p, _lib.c_int, _lib.c_ll, _lib.c_float
        _lib.declare(lib, "tnnb_muon_momentum", [p, p, p, p, i, l, f, i, f, p, i, p])
        _lib.declare(lib, "tnnb_muon_apply", [p, p, p, p, i, l, f, f, f, p, i, p])
        _lib.declare(lib, "tnnb_adam_pieces", [p, p, p, p, p, p, i, l, l, f, f, f, f, f, f, f, f, f, p, p, p])
        _MUON_DECLARED = True
    return lib


class MatrixGroup:
    """Equal matrices inside the flat buffers of a graph: ``offsets`` (elements) of ``[m, n]`` matrices. ``device``: where the buffers
    lie."""

    def __init__(self, m: int, n: int, offsets: Sequence[int], device):
        self.m, self.n, self.offsets = int(m), int(n), [int(o) for o in offsets]
        if self.m <= 0 or self.n <= 0 or not self.offsets:
            raise ValueError(f"{len(self.offsets)} matrices of {m} x {n}")
        self.size = self.m * self.n
        order = sorted(self.offsets)
        if any(b - a < self.size for a, b in zip(order, order[1:])):
            raise ValueError(f"matrices of {m} x {n} at {order} overlap")
        self.wide = int(self.size % 4 == 0 and all(o % 4 == 0 for o in self.offsets))
        self.table = torch.tensor(self.offsets, dtype=torch.int64, device=device)

    def check(self, flat: torch.Tensor, what: str) -> None:
        if flat.device != self.table.device:
            raise ValueError(f"{what} on {flat.device}, the matrices' places on {self.table.device}")
        if flat.dim() != 1 or not flat.is_contiguous() or min(self.offsets) < 0 or max(self.offsets) + self.size > flat.numel():
            raise ValueError(f"matrices of {self.m} x {self.n} do not lie in {what} of {tuple(flat.shape)}")


def muon_momentum(grads: torch.Tensor, group: MatrixGroup, buffer: torch.Tensor, momentum: float, nesterov: bool = True,
                  gscale: float = 1.0, hyper=None) -> torch.Tensor:
    """``buffer <- momentum * buffer + (1 - momentum) * g`` for the group's matrices of the flat fp32 ``grads``; returns the
    update ``[count, m, n]`` (fp32): the buffer, or with ``nesterov`` once more mixed with the gradient."""
    count = len(group.offsets)
    group.check(grads, "the gradients")
    if tuple(buffer.shape) != (count, group.m, group.n) or buffer.dtype != torch.float32 or grads.dtype != torch.float32 \
            or not buffer.is_contiguous() or buffer.device != grads.device:
        raise ValueError(f"momentum buffer {tuple(buffer.shape)} of {buffer.dtype} for {count} matrices of {group.m} x {group.n}")
    if grads.is_cuda:
        with _lib.device_of(grads):
            u = torch.empty_like(buffer)
            for i in range(0, count, 65535):
                k = min(65535, count - i)
                rc = _muon_library().tnnb_muon_momentum(grads, group.table[i:], buffer[i:], u[i:], k, group.size, momentum, int(nesterov), gscale,
                                                        hyper, group.wide, _lib.raw_stream())
                _lib.check_rc(rc, "muon_momentum")
                LAUNCHES["count"] += 1
        return u
    g = torch.stack([grads[o:o + group.size] for o in group.offsets]).view_as(buffer) * (gscale if hyper is None else hyper[3])
    buffer.mul_(momentum).add_(g * (1 - momentum))
    return buffer * momentum + g * (1 - momentum) if nesterov else buffer.clone()


def muon_apply(master: torch.Tensor, low, group: MatrixGroup, update: torch.Tensor, lr: float, factor: float, decay: float = 0.0,
               hyper=None) -> None:
    """``w <- w - lr * (factor * update + decay * w)`` for the group's matrices of the flat fp32 ``master``, and their rounded values into
    ``low`` (bf16, or None)."""
    count = len(group.offsets)
    group.check(master, "the weights")
    if update.numel() != count * group.size or update.dtype != torch.bfloat16 or not update.is_contiguous() \
            or master.dtype != torch.float32 or update.device != master.device:
        raise ValueError(f"update {tuple(update.shape)} of {update.dtype} for {count} matrices of {group.m} x {group.n}")
    if low is not None and (low.shape != master.shape or low.dtype != torch.bfloat16 or low.device != master.device):
        raise ValueError(f"compute copy {tuple(low.shape)} of {low.dtype} beside weights {tuple(master.shape)}")
    if low is not None and not low.is_contiguous():
        raise ValueError("a compute copy with gaps")
    update = update.view(count, -1)
    if master.is_cuda:
        with _lib.device_of(master):
            for i in range(0, count, 65535):
                k = min(65535, count - i)
                rc = _muon_library().tnnb_muon_apply(master, low, group.table[i:], update[i:], k, group.size, lr, factor, decay, hyper, group.wide,
                                                     _lib.raw_stream())
                _lib.check_rc(rc, "muon_apply")
                LAUNCHES["count"] += 1
        return
    rate = lr if hyper is None else hyper[0]
    for o, u in zip(group.offsets, update):
        w = master[o:o + group.size]
        w.sub_(rate * (factor * u.float() + decay * w))
        if low is not None:
            low[o:o + group.size].copy_(w)


def adam_pieces(master: torch.Tensor, low, grads: torch.Tensor, m: torch.Tensor, v: torch.Tensor, pieces: torch.Tensor, lr: float, b1: float,
                b2: float, eps: float, wd: float, step: int, gscale: float = 1.0, lr_ratio: float = 1.0, hyper=None) -> None:
    """:func:`raw.adam_step` over pieces of the flat buffers: ``pieces`` int64 ``[count, 3]``, on the buffers' device: offset, length and
    place in the packed moments ``m``, ``v``; no element in two pieces. A piece that does not lie in the buffers raises ``ValueError`` on CPU; on
    CUDA it is left out and recorded (``_lib.check_status``)."""
    for t, what in ((master, "weights"), (grads, "gradients"), (m, "moments"), (v, "moments")):
        if t.dtype != torch.float32 or t.dim() != 1 or not t.is_contiguous() or t.device != master.device:
            raise ValueError(f"{what} {tuple(t.shape)} of {t.dtype} on {t.device}: packed fp32 on {master.device} expected")
    if pieces.dim() != 2 or pieces.shape[1] != 3 or pieces.dtype != torch.int64 or pieces.device != master.device or not pieces.is_contiguous():
        raise ValueError(f"pieces {tuple(pieces.shape)} of {pieces.dtype} on {pieces.device}: int64 [count, 3] on {master.device} expected")
    if grads.shape != master.shape or m.shape != v.shape or (low is not None and (low.shape != master.shape or low.device != master.device)) \
            or (low is not None and master.is_cuda and (low.dtype != torch.bfloat16 or not low.is_contiguous())):
        raise ValueError("weights, gradients and compute copy, or the moments, differ in shape, or the copy is not packed bf16")
    bc1, bc2 = 1 - b1 ** step, 1 - b2 ** step
    if master.is_cuda:
        with _lib.device_of(master):
            rc = _muon_library().tnnb_adam_pieces(master, low, grads, m, v, pieces, pieces.shape[0], master.numel(), m.numel(), lr, b1, b2, eps, wd,
                                                  bc1, bc2, gscale, lr_ratio, hyper, _lib.status_addr(master.device), _lib.raw_stream())
            _lib.check_rc(rc, "adam_pieces")
            LAUNCHES["count"] += 1
        return
    if hyper is not None:
        lr, bc1, bc2, gscale = (float(x) for x in hyper)
    rate = lr * lr_ratio
    places = pieces.tolist()
    for at, n, st in places:
        if min(at, n, st) < 0 or at + n > master.numel() or st + n > m.numel():
            raise ValueError(f"a piece of {n} elements at {at}, its state at {st}: {master.numel()} weights, {m.numel()} moments")
    for at, n, st in places:
        g = grads[at:at + n].float() * gscale
        mi, vi, w = m[st:st + n], v[st:st + n], master[at:at + n]
        mi.mul_(b1).add_(g, alpha=1 - b1)
        vi.mul_(b2).addcmul_(g, g, value=1 - b2)
        w.sub_(rate * (mi / bc1) / (torch.sqrt(vi / bc2) + eps) + wd * rate * w)
        if low is not None:
            low[at:at + n].copy_(w.to(low.dtype))
