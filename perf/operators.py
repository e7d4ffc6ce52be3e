"""The operators around a language model's blocks, case by case: plain forms and the framework's kernels.

* ``embed``      rows of a token table, scaled, for given ids.
* ``embed_grad`` the table's gradient: the rows of every token's gradient added up per token.
* ``score``      log probabilities of given tokens with the entropy of each row's distribution and its top alternatives.
* ``score_grad`` the same as a training step meets it: log probabilities and entropies, and the gradient of the logits.
* ``orthogonalize`` the update of weight matrices by Newton-Schulz products, X <- a X + (b A + c A^2) X with A = X X^T.

``run`` computes them with elementary torch operations while ``own`` is false and through the framework's entry points
while it is true. ``exact`` is the definition in 64 bits, written apart from ``run``.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
NS_A, NS_B, NS_C, NS_EPS = 3.4445, -4.7750, 2.0315, 1e-7
IGNORED = -100  # the label of a position that counts for nothing


def listed():
    return [
        # one token for each of 16 requests that are being generated: all latency
        {"name": "embed_decode", "op": "embed", "tokens": 16, "vocab": 50257, "width": 768, "dtype": "bf16", "pad": False},
        # a batch of prompts or of training sequences, 16 x 1024, in front of the first block
        {"name": "embed_batch", "op": "embed", "tokens": 16384, "vocab": 50257, "width": 1024, "dtype": "bf16", "pad": True},
        # the table's gradient in a training step of 8 x 1024 tokens
        {"name": "embed_grad_batch", "op": "embed_grad", "tokens": 8192, "vocab": 50257, "width": 768, "dtype": "bf16", "pad": False},
        # long ragged batch with padding in it, fp32 training, a width that is no whole number of vectors
        {"name": "embed_grad_ragged", "op": "embed_grad", "tokens": 50001, "vocab": 32003, "width": 1001, "dtype": "fp32", "pad": True},
        # log probabilities and alternatives of one new token for each of eight requests
        {"name": "score_decode", "op": "score", "rows": 8, "vocab": 50257, "top": 20, "dtype": "bf16", "masked": False},
        # a text scored under the model: perplexity, evaluation of answers (8 x 1024 positions)
        {"name": "score_text", "op": "score", "rows": 8192, "vocab": 50257, "top": 5, "dtype": "bf16", "masked": False},
        # constrained generation: fp32 logits with tokens ruled out, some rows with none left, padding among the labels
        {"name": "score_masked", "op": "score", "rows": 999, "vocab": 128001, "top": 8, "dtype": "fp32", "masked": True},
        # a step that trains on log probabilities and entropies of the tokens that were sampled (4 x 1024 positions)
        {"name": "score_grad_batch", "op": "score_grad", "rows": 4096, "vocab": 50257, "top": 0, "dtype": "bf16", "masked": False},
        # the update of a single square projection
        {"name": "ortho_one", "op": "orthogonalize", "count": 1, "rows": 768, "cols": 768, "dtype": "fp32"},
        # the packed q, k, v projections of twelve blocks
        {"name": "ortho_qkv", "op": "orthogonalize", "count": 12, "rows": 2304, "cols": 768, "dtype": "fp32"},
        # the second MLP matrices of eight wider blocks, from bf16 momentum
        {"name": "ortho_wide", "op": "orthogonalize", "count": 8, "rows": 1280, "cols": 5120, "dtype": "bf16"},
        # convolution filters as matrices: odd extents, many small ones
        {"name": "ortho_odd", "op": "orthogonalize", "count": 9, "rows": 321, "cols": 1155, "dtype": "fp32"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even in its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "score", "score", "score_grad", "orthogonalize", "orthogonalize"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("embed", "embed_grad"):
        width = _spread(rng, 8, 2048)
        if rng.random() < 0.5:
            width = (width + 7) // 8 * 8
        most = 60_000_000 // width  # 240 MB of fp32 gradient and as much of table at most
        return {"op": op, "tokens": _spread(rng, 1, min(65536, most)), "vocab": _spread(rng, 100, min(130000, most)), "width": width,
                "dtype": dtype, "pad": rng.random() < 0.5}
    if op in ("score", "score_grad"):
        vocab = _spread(rng, 100, 160000)
        most = min(8192, 100_000_000 // vocab)
        return {"op": op, "rows": _spread(rng, 1, most), "vocab": vocab, "top": rng.randint(0, 32) if op == "score" else 0,
                "dtype": dtype, "masked": rng.random() < 0.5}
    rows, cols = _spread(rng, 16, 2048), _spread(rng, 16, 4096)
    low = min(rows, cols)
    flops = 10 * low * (2 * rows * cols + low * low)
    return {"op": op, "count": _spread(rng, 1, max(1, min(24, 400_000_000_000 // flops))), "rows": rows, "cols": cols, "dtype": dtype}


def _zipf(n, vocab, gen):
    """Ids whose frequency falls with their number, as in text."""
    u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)).long() - 1).clamp_(0, vocab - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] in ("embed", "embed_grad"):
        n, vocab, width = case["tokens"], case["vocab"], case["width"]
        ids = _zipf(n, vocab, gen)
        state = {"case": case, "ids": ids, "scale": math.sqrt(width), "padding": None, "vocab": vocab}
        if case["pad"]:  # sequences of unequal length: a fifth of the positions are padding
            state["padding"] = vocab - 1
            ids[torch.rand(n, device="cuda", generator=gen) < 0.2] = vocab - 1
        if case["op"] == "embed":
            state["table"] = (normal(vocab, width) / math.sqrt(width)).to(dtype)
        else:
            state["dy"] = (normal(n, width) * 1e-2).to(dtype)
        return state
    if case["op"] in ("score", "score_grad"):
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab)
        logits.mul_(2.0).sub_(torch.log(torch.arange(1, vocab + 1, device="cuda", dtype=torch.float32)))
        logits = logits.to(dtype)
        tokens = _zipf(rows, vocab, gen)
        if case["masked"]:
            logits[:, torch.rand(vocab, device="cuda", generator=gen) < 0.3] = -math.inf
            lowest = vocab // 3  # ruled out by the type's lowest value instead
            logits[:, lowest] = torch.finfo(dtype).min
            tokens[tokens == lowest] = 0
            tokens[torch.rand(rows, device="cuda", generator=gen) < 0.1] = IGNORED
            logits[rows // 2] = -math.inf  # nothing left
        state = {"case": case, "logits": logits, "tokens": tokens, "temperature": 0.8}
        if case["op"] == "score_grad":
            logits.requires_grad_()
            state["g_log"] = normal(rows) / rows
            state["g_ent"] = torch.full((rows,), -0.01 / rows, device="cuda")
        return state
    count, rows, cols = case["count"], case["rows"], case["cols"]
    # gradients of linear layers, averaged over steps: products of few tokens' signals of uneven strength, and noise
    few = 128
    out = normal(count, few, rows) * torch.exp(normal(count, 1, rows))
    inp = normal(count, few, cols) * torch.exp(0.5 * normal(count, 1, cols)) + normal(count, 1, cols)
    g = out.transpose(1, 2) @ inp
    g.mul_(1e-3 / few)
    g.add_(normal(count, rows, cols), alpha=2e-5)
    return {"case": case, "g": g.to(dtype)}


def _own(state):
    from tnn_b200.ops import functional as F
    from tnn_b200.ops import raw

    op = state["case"]["op"]
    if op == "embed":
        return F.embedding(state["ids"], state["table"], scale=state["scale"], padding_idx=state["padding"])
    if op == "embed_grad":
        return raw.embedding_grad(state["ids"], state["dy"], state["vocab"], scale=state["scale"], padding_idx=state["padding"])
    if op == "score":
        r = F.token_log_probs(state["logits"], state["tokens"], top_k=state["case"]["top"], temperature=state["temperature"])
        return list(r) if state["case"]["top"] else [r.log_probs, r.entropy]
    if op == "score_grad":
        r = F.token_log_probs(state["logits"], state["tokens"], temperature=state["temperature"])
        (d,) = torch.autograd.grad((r.log_probs, r.entropy), (state["logits"],), (state["g_log"], state["g_ent"]))
        return [r.log_probs.detach(), r.entropy.detach(), d]
    return raw.newton_schulz(state["g"])


def _plain_rows(z, tokens, temperature):
    """Log probabilities of all tokens, and of the given ones, and entropies, in the type of ``z``. A row without any token
    left has probability nowhere: its log probabilities are -inf and its entropy 0."""
    x = z / temperature
    top = x.max(1, keepdim=True).values
    dead = torch.isneginf(top)
    e = torch.exp(x - torch.where(dead, torch.zeros_like(top), top))
    lse = torch.where(dead, top, top + torch.log(e.sum(1, keepdim=True)))
    logp = torch.where(torch.isneginf(x), x, x - torch.where(dead, torch.zeros_like(lse), lse))
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    given = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    return logp, p, plogp, torch.where(tokens == IGNORED, torch.zeros_like(given), given), -plogp.sum(1)


@torch.no_grad()
def run(state):
    case = state["case"]
    if own:
        with torch.set_grad_enabled(case["op"] == "score_grad"):
            return _own(state)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "embed":
        y = state["table"][state["ids"]].float() * state["scale"]
        if state["padding"] is not None:
            y.mul_((state["ids"] != state["padding"])[:, None])
        return y.to(dtype)
    if case["op"] == "embed_grad":
        dy = state["dy"].float()
        if state["padding"] is not None:
            dy = dy * (state["ids"] != state["padding"])[:, None]
        d = torch.zeros(case["vocab"], case["width"], device=dy.device)
        d.index_add_(0, state["ids"], dy)
        return d.mul_(state["scale"]).to(dtype)
    if case["op"] in ("score", "score_grad"):
        z, tokens = state["logits"].float(), state["tokens"]
        logp, p, plogp, given, entropy = _plain_rows(z, tokens, state["temperature"])
        if case["op"] == "score":
            if not case["top"]:
                return [given, entropy]
            index = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            return [given, entropy, logp.gather(1, index), index]
        counts = (tokens != IGNORED) & ~torch.isneginf(z).all(1)
        g = torch.where(counts, state["g_log"], torch.zeros_like(state["g_log"]))[:, None]
        d = -p * g - state["g_ent"][:, None] * (plogp + p * entropy[:, None])
        d.scatter_add_(1, tokens.clamp(min=0)[:, None], g)
        return [given, entropy, d.div_(state["temperature"]).to(dtype)]
    x = state["g"].float()
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + NS_EPS)
    tall = case["rows"] > case["cols"]
    if tall:
        x = x.transpose(1, 2)
    for _ in range(5):
        a = x @ x.transpose(1, 2)
        x = NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x
    if tall:
        x = x.transpose(1, 2)
    return x.to(torch.bfloat16).contiguous()


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "embed":  # ids, each row that is named, the output
        return {"bytes": 8 * case["tokens"] + (min(case["tokens"], case["vocab"]) + case["tokens"]) * case["width"] * size,
                "flops": case["tokens"] * case["width"]}
    if case["op"] == "embed_grad":  # ids, the gradient of each position, the whole table's
        return {"bytes": 8 * case["tokens"] + (case["tokens"] + case["vocab"]) * case["width"] * size,
                "flops": 2 * case["tokens"] * case["width"]}
    if case["op"] == "score":
        return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 12 * case["top"]), "flops": 5 * case["rows"] * case["vocab"]}
    if case["op"] == "score_grad":  # the logits are needed twice, but the second time need not come from memory: once
        return {"bytes": case["rows"] * (2 * case["vocab"] * size + 24), "flops": 10 * case["rows"] * case["vocab"]}
    low, high = sorted((case["rows"], case["cols"]))
    # of the two symmetric products half the elements
    flops = 5 * case["count"] * (low * low * high + low ** 3 + 2 * low * low * high)
    return {"bytes": case["count"] * low * high * (size + 2), "flops": flops}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "embed":
        keep = torch.ones_like(s["ids"]) if s["padding"] is None else (s["ids"] != s["padding"]).long()
        return torch.index_select(s["table"], 0, s["ids"]).to(f64) * (keep * s["scale"])[:, None]
    if case["op"] == "embed_grad":
        ids = s["ids"]
        use = torch.arange(ids.numel(), device=ids.device)
        if s["padding"] is not None:
            use = use[ids != s["padding"]]
        order = use[torch.argsort(ids[use], stable=True)]
        out = torch.zeros(case["vocab"], case["width"], dtype=f64, device=ids.device)
        if order.numel():  # differences of running sums between the ends of each token's run
            rows = ids[order]
            last = torch.cat([rows[1:] != rows[:-1], torch.ones(1, dtype=torch.bool, device=ids.device)]).nonzero()[:, 0]
            total = torch.cumsum(s["dy"][order].to(f64), 0)[last]
            out[rows[last]] = torch.diff(total, dim=0, prepend=torch.zeros_like(total[:1])) * s["scale"]
        return out
    if case["op"] in ("score", "score_grad"):
        parts = []
        step = max(1, 64_000_000 // case["vocab"])
        for r in range(0, case["rows"], step):
            z = s["logits"][r:r + step].detach().to(f64)
            label = s["tokens"][r:r + step]
            logp = torch.log_softmax(z / s["temperature"], 1)
            none = (z == -math.inf).all(1)
            logp[none] = -math.inf
            entropy = torch.special.entr(logp.exp()).sum(1)
            counted = label != IGNORED
            at = torch.where(counted, label, 0)
            line = torch.arange(z.shape[0], device=z.device)
            given = torch.where(counted, logp[line, at], 0.0)
            if case["op"] == "score":
                part = [given, entropy]
                if case["top"]:
                    top = z.sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
                    part += [logp[line[:, None], top], top]
            else:
                g, h = s["g_log"][r:r + step].to(f64) * (counted & ~none), s["g_ent"][r:r + step].to(f64)
                p = logp.exp()
                d = p * -g[:, None] + h[:, None] * (torch.special.entr(p) - p * entropy[:, None])
                d[line, at] += g
                part = [given, entropy, d / s["temperature"]]
            parts.append(part)
        return [torch.cat(column) for column in zip(*parts)]
    y = s["g"].to(f64)
    y = y / (torch.linalg.matrix_norm(y)[:, None, None] + NS_EPS)
    for _ in range(5):
        if case["rows"] <= case["cols"]:
            gram = torch.bmm(y, y.mT)
            y = NS_A * y + torch.bmm(NS_B * gram + NS_C * torch.bmm(gram, gram), y)
        else:
            gram = torch.bmm(y.mT, y)
            y = NS_A * y + torch.bmm(y, NS_B * gram + NS_C * torch.bmm(gram, gram))
    return y
