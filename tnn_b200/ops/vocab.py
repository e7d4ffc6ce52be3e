"""The two ends of a language model, where its width meets the vocabulary: token embedding with scaling and its gradient
by sorted tokens (csrc/kernels/embedding.cu), log probabilities of given tokens with entropy and top alternatives
(csrc/kernels/token_logprob.cu).

CUDA tensors of bf16, fp16 and fp32 run the kernels; CPU tensors the same formulas in torch (fp32, or fp64 for fp64).
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .gemm import LAUNCHES

MAX_TOP = 32  # alternatives per row
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NO_ID = -(1 << 63)  # an id that no table has
_MAX_WIDTH = 1 << 30  # columns of a table: the kernels count them in 32 bits
_LOG2E = 1.4426950408889634
_DECLARED = False


_LIBRARY = None


def _library():
    global _DECLARED, _LIBRARY
    if _LIBRARY is not None:
        return _LIBRARY
    lib = _lib.load()
    if not _DECLARED:
        p, i, l, f = _lib.c_void_p, _lib.c_int, _lib.c_ll, _lib.c_float
        _lib.declare(lib, "tnnb_embed_lookup", [p, i, p, l, p, l, i, l, l, f, i, p])
        _lib.declare(lib, "tnnb_embed_grad", [p, i, p, l, p, p, p, p, p, p, i, i, l, l, f, i, i, i, i, p])
        _lib.declare(lib, "tnnb_token_logprob", [p, l, p, i, p, p, p, p, p, l, i, i, f, l, i, p])
        _lib.declare(lib, "tnnb_token_logprob_grad", [p, l, p, l, p, i, p, p, p, p, l, i, f, f, l, i, p])
        _DECLARED = True
    _LIBRARY = lib
    return lib


def _type_code(t: torch.Tensor, what: str) -> int:
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} is {t.dtype}; the kernels take bfloat16, float16 and float32")
    return code


def _whole(t: torch.Tensor, like: torch.Tensor, what: str) -> torch.Tensor:
    """Integer ids, packed, on ``like``'s device."""
    if t.dtype is not torch.int64 and t.dtype is not torch.int32:
        raise TypeError(f"{what} is {t.dtype}; int64 or int32 expected")
    if t.device != like.device:
        raise ValueError(f"{what} is on {t.device}, not on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _id(value: int) -> int:
    """A padding index or ignored token as the kernels compare it: one beyond 64 bits is no id's."""
    value = int(value)
    return value if _NO_ID < value < -_NO_ID else _NO_ID


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """``[rows, width]`` with a unit inner stride and rows that do not overlap."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if t.is_contiguous():
        return t
    return t if (t.stride(1) == 1 or width == 1) and (t.shape[0] < 2 or t.stride(0) >= width) else t.contiguous()


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors overlap."""
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()) for t in (a, b))
    return a0 < b1 and b0 < a1


def _new(like: torch.Tensor, dtype, *sizes: int) -> torch.Tensor:
    return torch.empty(sizes, dtype=dtype, device=like.device)  # (_lib.empty takes eight dimensions)


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]  # the stride of a single row means nothing


# ------------------------------------------------------------------------------------------------------- embedding
def embedding_lookup(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[ids]``, shape ``[*ids.shape, width]``: the product in fp32, rounded once to the table's type. Positions
    whose id is ``padding_idx`` are zero; an id outside the table reads row 0, like :func:`raw.embedding_fwd`. No derivative on CUDA:
    :func:`functional.embedding` has one."""
    if table.dim() != 2 or not table.is_floating_point():
        raise ValueError(f"embedding table {tuple(table.shape)} of {table.dtype}: a floating-point matrix expected")
    rows, width = table.shape
    flat = _whole(ids, table, "ids")
    n = flat.numel()
    if n and (rows == 0 or width == 0):
        raise ValueError(f"embedding table {tuple(table.shape)} is empty")
    if width > _MAX_WIDTH:
        raise ValueError(f"rows of {width} elements: at most {_MAX_WIDTH} are supported")
    pad = _NO_ID if padding_idx is None else _id(padding_idx)
    if table.is_cuda:
        code = _type_code(table, "embedding table")
        table = _rows(table, width)
        with _lib.device_of(table):
            out = _lib.empty(table, *ids.shape, width) if ids.dim() < 8 else _new(table, table.dtype, *ids.shape, width)
            if n:
                rc = _library().tnnb_embed_lookup(flat, flat.dtype is torch.int64, table.data_ptr(), max(_pitch(table), width), out, n, width, rows, pad,
                                                  float(scale), code, _lib.raw_stream())
                _lib.check_rc(rc, "embedding_lookup")
                LAUNCHES["count"] += 1
        return out
    flat = flat.reshape(-1).long()  # (compared as 32 bits, an index beyond them is cut off: no padding index was id 0)
    safe = torch.where((flat < 0) | (flat >= rows), torch.zeros_like(flat), flat)
    wide = torch.promote_types(table.dtype, torch.float32)
    out = table[safe].to(wide) * scale
    out = torch.where((flat == pad)[:, None], torch.zeros_like(out), out)
    return out.to(table.dtype).view(*ids.shape, width)


_FEW = 128  # positions whose gradient is one kernel without workspaces (embedding.cu's EMBED_FEW)


def _chunk(n: int) -> int:
    """Sorted positions per CTA of the gradient's sums: enough CTAs for the SMs (148, several on each), and no more parts of tokens
    that lie in several chunks than that takes. Us of the whole gradient with 16, 32, 64 and 128 (text-like ids): 1000 x 768 bf16 23.0*, 23.0,
    30.4, 43.4; 8192 x 768 30.0*, 27.6, 33.8, 47.8; 16384 x 1024 48.1*, 43.7, 45.5, 59.6; 20000 x 1001 fp32 65.4, 59.0*, 65.2, 84.9; 50001 x 1001 fp32 109.9, 99.1,
    104.9*, 105.0; 65536 x 768 bf16 92.8, 78.6, 75.1*, 71.7; 200000 x 768 234.5, 188.7, 170.5, 175.2* (* the one taken)."""
    chunk = 16
    while chunk < 128 and n > 1024 * chunk:
        chunk *= 2
    return chunk


def embedding_grad(ids: torch.Tensor, dy: torch.Tensor, rows: int, scale: float = 1.0, padding_idx: Optional[int] = None,
                   out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """Gradient of :func:`embedding_lookup` with respect to a table of ``rows`` rows: ``out[v] = scale * sum of dy over the
    positions whose id is v``. The sums are fp32 and rounded once; their order depends on the ids alone, so equal inputs give
    equal bits. ``out``: ``[rows, width]``, packed, of ``dy``'s type or fp32 (default: a new one of ``dy``'s type), every row of which
    is written; with ``accumulate`` (fp32) the sums are added to it instead."""
    rows = int(rows)
    if dy.dim() < 1 or dy.shape[:-1] != ids.shape or not dy.is_floating_point():
        raise ValueError(f"dy {tuple(dy.shape)} of {dy.dtype} does not belong to ids {tuple(ids.shape)}")
    width = dy.shape[-1]
    if rows <= 0 or width == 0:
        raise ValueError(f"the gradient of a table of {rows} rows of {width} elements is empty")
    flat = _whole(ids, dy, "ids")
    n = flat.numel()
    if n >= 1 << 30 or rows > 1 << 24 or width > _MAX_WIDTH:
        raise ValueError(f"{n} positions, {rows} rows of {width} elements: fewer than 2^30, at most 2^24 of at most {_MAX_WIDTH} are supported")
    if accumulate and out is None:
        raise ValueError("accumulate needs an output to add to")
    if out is not None:
        if tuple(out.shape) != (rows, width) or not out.is_contiguous() or out.device != dy.device:
            raise ValueError(f"out {tuple(out.shape)} on {out.device}: a packed [{rows}, {width}] on {dy.device} expected")
        if out.dtype not in ((torch.float32,) if accumulate else (dy.dtype, torch.float32)):
            raise TypeError(f"out is {out.dtype} for gradients of {dy.dtype}" + (" that are added up in fp32" if accumulate else ""))
    pad = _NO_ID if padding_idx is None else _id(padding_idx)
    if dy.is_cuda:
        code = _type_code(dy, "dy")
        dy2 = _rows(dy, width)
        with _lib.device_of(dy2):
            if out is None:
                out = _lib.empty(dy2, rows, width)
            elif n and _share_memory(out, dy2):
                dy2 = dy2.clone(memory_format=torch.contiguous_format)  # rows are written while others are still read
            pitch = max(_pitch(dy2), width) if n else width
            if n <= _FEW:
                rc = _library().tnnb_embed_grad(flat, flat.dtype is torch.int64, dy2, pitch, out, None, None, None, None, None, n, width, rows, pad,
                                                float(scale), code, _TYPES[out.dtype], int(accumulate), 16, _lib.raw_stream())
                _lib.check_rc(rc, "embedding_grad")
                LAUNCHES["count"] += 1 if n else 0
                return out
            chunk = _chunk(n)
            # where each position belongs, sorted positions and their tokens, where each row's begin; partial sums of tokens in several chunks
            n4 = (n + 3) // 4 * 4
            ints = _lib.empty(dy2, torch.int32, n4 + 2 * n + rows + rows // 256 + 129)
            parts = _lib.empty(dy2, torch.float32, 2 * ((n + chunk - 1) // chunk) * width)
            base = ints.data_ptr()
            rc = _library().tnnb_embed_grad(flat, flat.dtype is torch.int64, dy2, pitch, out, base, base + 4 * n4, base + 4 * (n4 + n),
                                            base + 4 * (n4 + 2 * n), parts, n, width, rows, pad, float(scale), code, _TYPES[out.dtype],
                                            int(accumulate), chunk, _lib.raw_stream())
            _lib.check_rc(rc, "embedding_grad")
            LAUNCHES["count"] += 4
        return out
    flat = flat.reshape(-1).long()  # (compared as 32 bits, an index beyond them is cut off: no padding index was id 0)
    safe = torch.where((flat < 0) | (flat >= rows), torch.zeros_like(flat), flat)
    g = dy.reshape(-1, width).to(torch.promote_types(dy.dtype, torch.float32))
    g = torch.where((flat == pad)[:, None], torch.zeros_like(g), g)
    total = torch.zeros(rows, width, dtype=g.dtype).index_add_(0, safe, g) * scale
    if out is None:
        return total.to(dy.dtype)
    return out.add_(total.to(out.dtype)) if accumulate else out.copy_(total.to(out.dtype))


# ------------------------------------------------------------------------------------------- token log probabilities
class TokenLogProbs(NamedTuple):
    log_probs: torch.Tensor      # [*rows] log probability of the given token
    entropy: torch.Tensor        # [*rows] of the row's distribution, in nats
    top_log_probs: torch.Tensor  # [*rows, top_k], descending
    top_indices: torch.Tensor    # [*rows, top_k] int64; of equal logits the lowest index comes first


def _check_rows(logits, tokens, top_k, temperature):
    shape = logits.shape
    if not shape or shape[:-1] != tokens.shape or not logits.is_floating_point():
        raise ValueError(f"logits {tuple(shape)} of {logits.dtype} do not belong to tokens {tuple(tokens.shape)}")
    V = shape[-1]
    if V == 0 or V >= 1 << 30:
        raise ValueError(f"a vocabulary of {V} tokens")
    if not 0 <= top_k <= min(MAX_TOP, V):
        raise ValueError(f"top_k {top_k}: 0 to {min(MAX_TOP, V)} alternatives of {V} tokens")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature {temperature}: 1e-6 to 1e6 are supported")
    return V


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0, temperature: float = 1.0, ignore_index: int = -100,
                    keep: Optional[dict] = None) -> TokenLogProbs:
    """Log probabilities of ``tokens`` (one per row of ``logits [*rows, V]``) under ``softmax(logits / temperature)``, each row's
    entropy and its ``top_k`` most likely tokens, in one pass over the logits; fp32 results.

    Positions of ``ignore_index`` get log probability 0 (their entropy and alternatives are those of their row). Any other token outside
    the vocabulary has log probability NaN. A row with nothing but -inf has log probability -inf and entropy 0; a NaN or +inf logit
    makes a row's results NaN (NaN sorts first, and the indices are those of the largest logits all the same). ``keep``: a dict that
    receives what :func:`token_log_probs_grad` needs, the entropies of the result among it (which have to stay as they are until then).
    No derivative on CUDA: :func:`functional.token_log_probs` has one."""
    top_k, temperature, ignore_index, shape = int(top_k), float(temperature), _id(ignore_index), tokens.shape
    V = _check_rows(logits, tokens, top_k, temperature)
    tok = _whole(tokens, logits, "tokens")
    z = _rows(logits, V)
    rows = z.shape[0]
    if logits.is_cuda:
        code = _type_code(logits, "logits")
        with _lib.device_of(z):
            f32 = torch.float32
            new = _lib.empty if len(shape) < 8 else _new
            lp, ent = new(z, f32, *shape), new(z, f32, *shape)
            top, idx = new(z, f32, *shape, top_k), new(z, torch.int64, *shape, top_k)
            stats = _lib.empty(z, f32, rows, 2) if keep is not None else None
            if rows:
                rc = _library().tnnb_token_logprob(z.data_ptr(), max(_pitch(z), V), tok, tok.dtype is torch.int64, lp, ent, top, idx, stats, rows, V, top_k,
                                                   _LOG2E / temperature, ignore_index, code, _lib.raw_stream())
                _lib.check_rc(rc, "token_log_probs")
                LAUNCHES["count"] += 1
        if keep is not None:
            keep.update(stats=stats, entropy=ent)
        return TokenLogProbs(lp, ent, top, idx)
    tok = tok.reshape(-1).long()
    wide = torch.promote_types(z.dtype, torch.float32)
    zf = z.to(wide)
    logp, p, plogp = _distribution(zf, temperature)
    known = (tok >= 0) & (tok < V)
    lp = logp.gather(1, torch.where(known, tok, torch.zeros_like(tok))[:, None])[:, 0]
    lp = torch.where(known, lp, torch.full_like(lp, math.nan))
    lp = torch.where(tok == ignore_index, torch.zeros_like(lp), lp)
    # explicit keys: torch orders -0 and 0 as equal, NaN above everything, which is the order wanted
    idx = torch.sort(zf, dim=1, descending=True, stable=True).indices[:, :top_k]
    top, ent = logp.gather(1, idx), (-plogp.sum(1)).clamp_min(0)
    if keep is not None:
        keep.update(stats=None, entropy=ent)
    return TokenLogProbs(lp.view(shape), ent.view(shape), top.view(*shape, top_k), idx.reshape(*shape, top_k))


def _distribution(z: torch.Tensor, temperature: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``log p``, ``p`` and ``p log p`` of every element, with the conventions of :func:`token_log_probs`."""
    m = z.max(1, keepdim=True).values
    dead = torch.isneginf(m)
    bad = torch.isnan(m) | torch.isposinf(m)
    # relative to the maximum before anything is rounded: beside a large one the sum's logarithm would be lost, and a quotient by the
    # temperature might overflow
    d = (z - torch.where(dead | bad, torch.zeros_like(m), m)) / temperature
    logp = torch.where(torch.isneginf(z), z, d - torch.log(torch.exp(d).sum(1, keepdim=True)))
    logp = torch.where(bad, torch.full_like(logp, math.nan), logp)
    p = torch.exp(logp)
    plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
    return logp, p, plogp


def _kept(t: Optional[torch.Tensor], size: int, z: torch.Tensor) -> bool:
    return t is not None and t.dtype is torch.float32 and t.numel() == size and t.device == z.device and t.is_contiguous()


def token_log_probs_grad(logits: torch.Tensor, tokens: torch.Tensor, kept: dict, g_log_probs: Optional[torch.Tensor],
                         g_entropy: Optional[torch.Tensor], temperature: float = 1.0, ignore_index: int = -100) -> torch.Tensor:
    """Gradient with respect to ``logits`` for gradients of the log probabilities and the entropies (None: zero). ``kept``: what the
    forward call left in its ``keep``. Rows without a distribution get zeros. The result has the shape of ``logits`` and, where the
    gaps between its rows are smaller than a row, the same gaps."""
    V = _check_rows(logits, tokens, 0, float(temperature))
    ignore_index = _id(ignore_index)
    tok = _whole(tokens, logits, "tokens")
    z = _rows(logits, V)
    rows = z.shape[0]

    def grad_of(g):
        if g is None:
            return None
        if g.numel() != rows or g.device != z.device:
            raise ValueError(f"a gradient of {g.numel()} values on {g.device} for {rows} rows on {z.device}")
        if g.dtype is torch.float32 and g.dim() == 1 and g.is_contiguous() and z.dtype is not torch.float64:
            return g
        return g.reshape(-1).to(torch.promote_types(z.dtype, torch.float32)).contiguous()

    g, h = grad_of(g_log_probs), grad_of(g_entropy)
    if logits.is_cuda:
        code = _type_code(logits, "logits")
        stats, entropy = kept["stats"], kept["entropy"]
        if not (_kept(stats, 2 * rows, z) and _kept(entropy, rows, z)):
            raise ValueError(f"the statistics that were kept do not belong to {rows} rows on {z.device}")
        with _lib.device_of(z):
            pitch = max(_pitch(z), V)
            # rows far apart (the last position of every sequence): not that much memory between those of the result, and the same
            # place within 16 bytes, so that rows of both share vectors
            out_pitch = pitch if pitch < 2 * V else V + (pitch - V) % 8
            dz = _lib.empty(z, rows, out_pitch)
            if out_pitch != V:
                dz = dz[:, :V]
            if rows:
                rc = _library().tnnb_token_logprob_grad(z.data_ptr(), pitch, dz, out_pitch, tok, tok.dtype is torch.int64, stats, entropy,
                                                        g, h, rows, V, _LOG2E / float(temperature), 1.0 / float(temperature),
                                                        ignore_index, code, _lib.raw_stream())
                _lib.check_rc(rc, "token_log_probs_grad")
                LAUNCHES["count"] += 1
        if logits.dim() == 2:
            return dz
        return dz.view(logits.shape) if out_pitch == V else dz.unflatten(0, logits.shape[:-1])
    entropy = kept["entropy"]
    if entropy is None or entropy.numel() != rows or entropy.device != z.device:
        raise ValueError(f"the entropies that were kept do not belong to {rows} rows on {z.device}")
    tok = tok.reshape(-1).long()
    zf = z.to(torch.promote_types(z.dtype, torch.float32))
    logp, p, plogp = _distribution(zf, float(temperature))
    dead = torch.isneginf(zf).all(1)
    nothing = torch.zeros(rows, dtype=zf.dtype)
    counts = (tok != ignore_index) & ~dead
    g = torch.where(counts, g, nothing) if g is not None else nothing
    h = torch.where(dead, nothing, h) if h is not None else nothing
    known = (tok >= 0) & (tok < V)
    g = torch.where((tok != ignore_index) & ~known, torch.full_like(g, math.nan), g)
    d = -p * g[:, None] - h[:, None] * (plogp + p * entropy.reshape(-1, 1))
    d.scatter_add_(1, torch.where(known, tok, torch.zeros_like(tok))[:, None], torch.where(known, g, nothing)[:, None])
    return torch.where(dead[:, None], torch.zeros_like(d), d / float(temperature)).to(logits.dtype).view(logits.shape)
