"""Definitions in 64 bits of the operators at a language model's vocabulary, and the inputs their tests share."""
import math

import torch


def ids_for(n, vocab, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":  # every position names the same token
        return torch.full((n,), vocab // 2, dtype=torch.int64)
    if kind == "zipf":
        return (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(vocab + 1)).long() - 1).clamp(0, vocab - 1)
    return torch.randint(0, vocab, (n,), generator=g)


def embedding64(ids, table, scale, padding_idx):
    safe = torch.where((ids < 0) | (ids >= table.shape[0]), 0, ids)
    y = table.double()[safe] * scale
    if padding_idx is not None:
        y[ids == padding_idx] = 0
    return y


def embedding_grad64(ids, dy, rows, scale, padding_idx):
    """(sums, sums of magnitudes, positions per row)"""
    safe = torch.where((ids < 0) | (ids >= rows), 0, ids)
    use = torch.ones_like(ids, dtype=torch.bool) if padding_idx is None else ids != padding_idx
    d = torch.zeros(rows, dy.shape[-1], dtype=torch.float64)
    mag, count = torch.zeros_like(d), torch.zeros(rows, dtype=torch.float64)
    for t in range(ids.numel()):
        if use[t]:
            d[safe[t]] += dy[t].double() * scale
            mag[safe[t]] += (dy[t].double() * scale).abs()
            count[safe[t]] += 1
    return d, mag, count


def logits_for(rows, vocab, dtype, kind, seed):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=g) * 2.5
    if kind == "masked":
        z[:, torch.rand(vocab, generator=g) < 0.4] = -math.inf
        if vocab > 2:
            z[:, 1] = torch.finfo(dtype).min
        z[rows // 2] = -math.inf
    elif kind == "few":  # all but two tokens of each row ruled out
        keep = torch.randint(0, vocab, (rows, 2), generator=g)
        z = torch.full_like(z, -math.inf).scatter(1, keep, z.gather(1, keep))
    elif kind == "equal":
        z = torch.zeros_like(z)
    elif kind == "coarse":  # many equal values, and both zeros
        z = z.round() * torch.where(torch.rand(rows, vocab, generator=g) < 0.5, 1.0, -1.0)
    elif kind == "rising":
        z = torch.arange(vocab).float().mul(8.0 / vocab).expand(rows, vocab).clone()
    elif kind == "peaked":
        z[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] = 60.0
    elif kind == "large":
        z = z * 40 + 900
    elif kind == "bad":  # not a number and +inf
        z[0, vocab // 3] = math.nan
        z[-1, vocab // 2] = math.inf
    return z.to(dtype)


def logprobs64(z, tokens, top_k, temperature, ignore_index):
    x = z.double() / temperature
    m = x.max(1).values
    dead, bad = torch.isneginf(m), torch.isnan(m) | torch.isposinf(m)
    logp = torch.log_softmax(x, 1)
    logp[dead] = -math.inf
    logp[bad] = math.nan
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    plogp[bad] = math.nan
    known = (tokens >= 0) & (tokens < z.shape[1])
    lp = logp.gather(1, torch.where(known, tokens, 0)[:, None])[:, 0]
    lp[~known] = math.nan
    lp[tokens == ignore_index] = 0
    idx = torch.sort(z.float(), dim=1, descending=True, stable=True).indices[:, :top_k]
    return lp, -plogp.sum(1), logp.gather(1, idx), idx, logp, p, plogp


def logprobs_grad64(z, tokens, g, h, temperature, ignore_index):
    """(gradient, the magnitudes of its terms added up)"""
    _, ent, _, _, logp, p, plogp = logprobs64(z, tokens, 0, temperature, ignore_index)
    dead = torch.isneginf(z).all(1)
    gg = torch.where((tokens == ignore_index) | dead, 0.0, g.double())[:, None]
    hh = torch.where(dead, 0.0, h.double())[:, None]
    d = -p * gg - hh * (plogp + p * ent[:, None])
    mag = p * gg.abs() + hh.abs() * (plogp.abs() + p * ent[:, None])
    at = tokens.clamp(min=0)[:, None]
    d.scatter_add_(1, at, gg)
    mag.scatter_add_(1, at, gg.abs())
    d[dead] = 0
    return d / temperature, mag / temperature
