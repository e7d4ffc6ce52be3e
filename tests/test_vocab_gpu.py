"""The embedding and token-log-probability kernels against their definitions in 64 bits."""
import math

import pytest
import torch

from tests._vocab_reference import embedding64, embedding_grad64, ids_for, logits_for, logprobs64, logprobs_grad64
from tnn_b200.ops import functional as F
from tnn_b200.ops import raw

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
# half a step below the smallest normal number (fp32 ones that small are flushed to zero: a whole one)
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def within(got, ref, tol, what=""):
    got, ref = got.double().cpu(), ref.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), what
    tol = (torch.zeros_like(ref) + tol)[fine]
    over = ((got[fine] - ref[fine]).abs() - tol)
    assert not bool((over > 0).any()), f"{what}: off by {float(over.max()):.3g} more than allowed, {int((over > 0).sum())} of {over.numel()}"


# ------------------------------------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 50, 8), (7, 300, 33), (64, 17, 768), (257, 1000, 1027), (1000, 40, 136)])
@pytest.mark.parametrize("padding", [None, 0])
def test_lookup(dtype, n, vocab, width, padding):
    ids = ids_for(n, vocab, "zipf", n + width)
    if n > 5:
        ids[2], ids[5] = vocab + 3, -1
    table = torch.randn(vocab, width, generator=torch.Generator().manual_seed(1)).to(dtype)
    for kind in (torch.int64, torch.int32):
        y = raw.embedding_lookup(ids.cuda().to(kind), table.cuda(), 3.3, padding)
        ref = embedding64(ids, table, 3.3, padding)
        # the scale rounded to fp32, the product in fp32, then the type
        within(y, ref, (HALF[dtype] + 2 * 2.0 ** -24) * ref.abs() + TINY[dtype])


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_of_strided_and_offset_tables(dtype):
    ids = ids_for(90, 60, "zipf", 3)
    wide = torch.randn(60, 100).to(dtype)
    for cut in (wide[:, :64], wide[:, 1:65], wide[:, 8:96], wide.t()[:50].t(), wide[::2, :40]):
        rows = cut.shape[0]
        at = ids % rows
        y = raw.embedding_lookup(at.view(9, 10).cuda(), wide.cuda().as_strided(cut.shape, cut.stride(), cut.storage_offset()), 1.0)
        assert y.shape == (9, 10, cut.shape[1]) and torch.equal(y.view(90, -1).cpu(), cut[at])


GRAD_SHAPES = [(1, 1, 1), (1, 50, 8), (15, 9, 33), (16, 300, 64), (17, 1, 8), (300, 1, 40), (257, 1000, 129), (3000, 700, 96), (20011, 5000, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,width", GRAD_SHAPES)
@pytest.mark.parametrize("kind", ["zipf", "one", "uniform"])
def test_embedding_gradient(dtype, n, vocab, width, kind):
    ids = ids_for(n, vocab, kind, n)
    if n > 15:
        ids[3], ids[15] = vocab + 3, -1
    padding = vocab - 1 if n % 2 else None
    dy = torch.randn(n, width, generator=torch.Generator().manual_seed(2)).to(dtype)
    ref, mag, count = embedding_grad64(ids, dy, vocab, 1.3, padding)
    # each of the additions and the product with the (rounded) scale is off by half a step of what has been added up so far
    summed = (count[:, None] + 2) * 2.0 ** -24 * mag
    for out_type in {dtype, torch.float32}:
        out = torch.full((vocab, width), math.nan, dtype=out_type, device="cuda")  # every element is written
        got = raw.embedding_grad(ids.cuda(), dy.cuda(), vocab, 1.3, padding, out)
        assert got is out
        within(got, ref, HALF[out_type] * (ref.abs() + summed) + summed + TINY[out_type], f"into {out_type}")
        again = raw.embedding_grad(ids.cuda().int(), dy.cuda(), vocab, 1.3, padding, torch.empty_like(out))
        assert torch.equal(got, again)  # no sum depends on who comes first
    base = torch.randn(vocab, width)
    acc = raw.embedding_grad(ids.cuda(), dy.cuda(), vocab, 1.3, padding, base.cuda(), accumulate=True)
    within(acc, ref + base.double(), summed + 2.0 ** -23 * (ref.abs() + base.abs().double()) + TINY[torch.float32], "added")
    untouched = count == 0
    assert torch.equal(acc.cpu()[untouched], base[untouched])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,width", [(2, 70001, 8), (31, 500, 1027), (33, 8, 2056), (127, 100, 300), (128, 700, 96), (129, 700, 96), (128, 3, 1030)])
@pytest.mark.parametrize("kind", ["zipf", "one", "uniform"])
def test_embedding_gradient_of_few_positions(dtype, n, vocab, width, kind):
    test_embedding_gradient(dtype, n, vocab, width, kind)


def test_embedding_gradient_of_views_and_large_vocabularies():
    n, vocab, width = 500, 200_003, 16  # more rows than two CTAs per SM hold at 512 each
    ids = ids_for(n, vocab, "uniform", 4)
    wide = torch.randn(n, 40).to(torch.bfloat16)
    for cut in (wide[:, :16], wide[:, 3:19], wide[:, ::2][:, :16], wide[:1, :16].expand(n, 16)):
        d = raw.embedding_grad(ids.cuda(), wide.cuda().as_strided(cut.shape, cut.stride(), cut.storage_offset()), vocab)
        ref, mag, _ = embedding_grad64(ids, cut, vocab, 1.0, None)
        within(d, ref, HALF[torch.bfloat16] * ref.abs() + 8 * 2.0 ** -24 * mag + TINY[torch.bfloat16])


# ------------------------------------------------------------------------------------------- token log probabilities
ROWS = [(1, 1), (1, 9), (3, 31), (5, 257), (2, 1000), (3, 8191), (1, 20003), (9, 50257), (300, 2051), (301, 8200), (2, 131072)]
KINDS = ["plain", "masked", "few", "equal", "coarse", "rising", "peaked", "large", "bad"]


def _tolerances(z, tokens, lp, ent, vocab, temperature):
    """Steps of 2^-24: each of a thread's four sums takes up to vocab / 256 terms one after the other (64 threads or more), then 8 + 8 + 8 joins; each exponent is off
    by half a step of itself and each exponential by four (the instruction's two, and the product it is taken of); log2(e) / T is
    rounded (relative to the exponent), the result is rounded. Rounding the maximum's exponent is common to all terms and cancels."""
    chain = vocab / 256 + 24 + 8
    m = z.double().masked_fill(torch.isinf(z) | torch.isnan(z), -1e4).max(1).values / temperature
    at = z.double().gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0] / temperature
    span = torch.where(torch.isfinite(at), (m - at).abs().clamp(max=1e5), 0.0)
    spread = torch.nan_to_num(ent) + 1  # mean distance of exponents from the maximum is at most log of the sum, this the scale of both
    logsum = math.log(vocab) + 1
    step = 2.0 ** -24
    tol_lp = step * (chain + 4 * (span + torch.nan_to_num(lp, neginf=0).abs()) + 2 * logsum)
    tol_ent = step * (4 * chain * (spread + logsum) + 4 * logsum)
    return tol_lp, tol_ent


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", ROWS)
@pytest.mark.parametrize("kind", KINDS)
def test_token_log_probs(dtype, rows, vocab, kind):
    z = logits_for(rows, vocab, dtype, kind, rows + vocab)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(7))
    if kind != "plain" and vocab > 2:
        tokens[tokens == 1] = 0  # holds the type's lowest value in masked rows: its quotient by the temperature exceeds fp32
    if rows > 4:
        tokens[1], tokens[4] = -100, vocab
    T = 0.8 if kind != "large" else 1.0
    top = min(vocab, {1: 1, 3: 5, 9: 20, 2: 32}.get(rows, 8))
    lp, ent, tv, ti, *_ = logprobs64(z, tokens, top, T, -100)
    r = raw.token_log_probs(z.cuda(), tokens.cuda(), top, T)
    assert torch.equal(r.top_indices.cpu(), ti), kind
    tol_lp, tol_ent = _tolerances(z, tokens, lp, ent, vocab, T)
    within(r.log_probs, lp, tol_lp, "log probability")
    within(r.entropy, ent, tol_ent, "entropy")
    live = torch.where(torch.isfinite(tv), tv, torch.zeros_like(tv)).abs()
    lowest = z.float().gather(1, ti) <= torch.finfo(dtype).min
    shown = torch.where(lowest & torch.isfinite(tv), r.top_log_probs.cpu().double(), tv)  # as for tokens == 1 above
    within(r.top_log_probs, shown, tol_lp.max() + 2.0 ** -22 * live, "alternatives")
    plain = raw.token_log_probs(z.cuda(), tokens.cuda().int(), 0, T)  # without alternatives: the same numbers
    assert torch.equal(plain.log_probs.nan_to_num(7), r.log_probs.nan_to_num(7)) and plain.top_indices.shape == (rows, 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_logits(dtype):
    wide = (torch.randn(40, 1040) * 3).to(dtype)
    for cut in (wide[:, :1000], wide[:, 3:1000], wide[::3, 8:1032], wide.t()[:700].t(), wide[:1].expand(40, 1040)):
        z = wide.cuda().as_strided(cut.shape, cut.stride(), cut.storage_offset()).requires_grad_()
        tokens = torch.arange(cut.shape[0]) * 7
        r = F.token_log_probs(z, tokens.cuda(), 4, 1.1)
        lp, ent, tv, ti, *_ = logprobs64(cut, tokens, 4, 1.1, -100)
        assert torch.equal(r.top_indices.cpu(), ti)
        tol_lp, tol_ent = _tolerances(cut, tokens, lp, ent, cut.shape[1], 1.1)
        within(r.log_probs.detach(), lp, tol_lp)
        within(r.entropy.detach(), ent, tol_ent)
        g, h = torch.randn(cut.shape[0]), torch.randn(cut.shape[0])
        (d,) = torch.autograd.grad((r.log_probs, r.entropy), (z,), (g.cuda(), h.cuda()))
        ref, mag = logprobs_grad64(cut, tokens, g, h, 1.1, -100)
        within(d, ref, HALF[dtype] * ref.abs() + 2.0 ** -24 * 200 * mag + TINY[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (2, 1000), (3, 8191), (9, 50257), (300, 2051)])
@pytest.mark.parametrize("kind", ["plain", "masked", "few", "equal", "peaked", "large"])
def test_token_log_probs_gradient(dtype, rows, vocab, kind):
    z = logits_for(rows, vocab, dtype, kind, rows + vocab)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(8))
    if rows > 4:
        tokens[1] = -100
    g, h = torch.randn(rows), torch.randn(rows)
    T = 0.8 if kind != "large" else 1.0
    zc = z.cuda().requires_grad_()
    r = F.token_log_probs(zc, tokens.cuda(), 0, T)
    (d,) = torch.autograd.grad((r.log_probs, r.entropy), (zc,), (g.cuda(), h.cuda()))
    ref, mag = logprobs_grad64(z, tokens, g, h, T, -100)
    # A probability is off by its exponent's error: the sum's (chain as in _tolerances), half a step of the exponent's terms (the
    # logit's and the maximum's, each rounded) and the exponential's own; every product with it and the entropy's error come on top.
    # A probability below 2^-126 is flushed to zero, and with it its terms g p and h p (log p + H), where |log p| < 88: at most
    # 2^-126 (|g| + |h| (88 + H)) / T are lost.
    size = torch.where(torch.isfinite(z), z.double().abs(), torch.zeros((), dtype=torch.float64)).clamp(max=2e3) / T
    steps = vocab / 256 + 40 + 4 * size + 4 * size.max(1, keepdim=True).values
    ent_off = _tolerances(z, tokens, torch.zeros(rows, dtype=torch.float64), logprobs64(z, tokens, 0, T, -100)[1], vocab, T)[1]
    p = logprobs64(z, tokens, 0, T, -100)[5]
    lost = 2.0 ** -126 * (g.abs() + h.abs() * (88 + math.log(vocab))).double()[:, None] / T
    tol = HALF[dtype] * ref.abs() + 2.0 ** -24 * steps * mag + p * (h.double().abs() * ent_off)[:, None] / T + lost + TINY[dtype]
    within(d, ref, tol, kind)


def test_bad_rows_have_no_gradient_numbers():
    z = logits_for(3, 40, torch.float32, "bad", 1).cuda().requires_grad_()
    r = F.token_log_probs(z, torch.tensor([1, 40, 2], device="cuda"))
    r.log_probs.sum().backward()
    assert bool(torch.isnan(z.grad).all())  # NaN, a token outside of the vocabulary, +inf


def test_one_gradient_only_and_3d():
    z = (torch.randn(2, 5, 333) * 2).to(torch.bfloat16)
    tokens = torch.randint(0, 333, (2, 5))
    for which in ("log_probs", "entropy"):
        zc = z.cuda().requires_grad_()
        getattr(F.token_log_probs(zc, tokens.cuda()), which).sum().backward()
        one, zero = torch.ones(10), torch.zeros(10)
        ref, mag = logprobs_grad64(z.view(10, 333), tokens.view(10), one if which == "log_probs" else zero,
                                   one if which == "entropy" else zero, 1.0, -100)
        within(zc.grad.view(10, 333), ref, HALF[torch.bfloat16] * ref.abs() + 2.0 ** -24 * 400 * mag + 1e-30)


def test_captured_and_replayed():
    """One graph over both directions, replayed on new inputs, against eager calls; on a side stream."""
    ids = ids_for(700, 900, "zipf", 1).cuda()
    table = torch.randn(900, 72, device="cuda", dtype=torch.bfloat16)
    dy = torch.randn(700, 72, device="cuda", dtype=torch.bfloat16)
    z = torch.randn(9, 9001, device="cuda", dtype=torch.bfloat16)
    tok = torch.randint(0, 9001, (9,), device="cuda")
    g = torch.randn(9, device="cuda")

    def work():
        keep = {}
        r = raw.token_log_probs(z, tok, 5, 1.0, keep=keep)
        return [raw.embedding_lookup(ids, table, 2.0), raw.embedding_grad(ids, dy, 900, 2.0), *r,
                raw.token_log_probs_grad(z, tok, keep, g, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = work()
    torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 2):
        ids.copy_(ids_for(700, 900, "zipf", seed + 10))
        z.copy_(torch.randn(9, 9001, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        got = [t.clone() for t in out]
        for a, b in zip(got, work()):
            assert torch.equal(a, b)


def test_refusals_on_the_gpu():
    from tests.test_vocab_cpu import _refusals

    for i, (error, call) in enumerate(_refusals("cuda")):
        with pytest.raises(error):
            call()
    z = torch.zeros(2, 8, device="cuda")
    with pytest.raises(ValueError):
        raw.token_log_probs(z, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        raw.token_log_probs(z.double(), torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError):
        raw.embedding_lookup(torch.zeros(2, dtype=torch.int64, device="cuda"), z.double())


def test_empty_batches():
    none = torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    assert raw.embedding_lookup(none, torch.zeros(3, 4, device="cuda")).shape == (2, 0, 4)
    assert torch.equal(raw.embedding_grad(none, torch.zeros(2, 0, 4, device="cuda"), 3).cpu(), torch.zeros(3, 4))
    r = raw.token_log_probs(torch.zeros(2, 0, 5, device="cuda"), none, 2)
    assert r.log_probs.shape == (2, 0) and r.top_indices.shape == (2, 0, 2)


def test_many_dimensions():
    ids = torch.arange(6, device="cuda").view(1, 1, 2, 1, 3, 1, 1, 1, 1)
    table = torch.randn(6, 5, device="cuda")
    assert torch.equal(raw.embedding_lookup(ids, table), table.view(1, 1, 2, 1, 3, 1, 1, 1, 1, 5))
    assert torch.equal(raw.embedding_grad(ids, table.view(*ids.shape, 5), 6), table)
    z = torch.randn(6, 9, device="cuda")
    keep, flat = {}, {}
    r, s = raw.token_log_probs(z.view(*ids.shape, 9), ids, 2, keep=keep), raw.token_log_probs(z, ids.view(6), 2, keep=flat)
    for a, b in zip(r, s):
        assert torch.equal(a.reshape(b.shape), b) and a.shape[:9] == ids.shape
    g = torch.randn(6, device="cuda")
    assert torch.equal(raw.token_log_probs_grad(z.view(*ids.shape, 9), ids, keep, g, g).view(6, 9),
                       raw.token_log_probs_grad(z, ids.view(6), flat, g, g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1000, 1003])
def test_gradient_of_the_last_positions(dtype, vocab):
    """Rows a whole sequence apart: the gradient leaves no such gaps."""
    z = torch.randn(5, 7, vocab).to(dtype)
    tokens, g, h = torch.randint(0, vocab, (5,)), torch.randn(5), torch.randn(5)
    keep = {}
    last = z.cuda()[:, -1]
    raw.token_log_probs(last, tokens.cuda(), keep=keep)
    d = raw.token_log_probs_grad(last, tokens.cuda(), keep, g.cuda(), h.cuda())
    assert d.untyped_storage().nbytes() <= 5 * (vocab + 8) * z.element_size()
    ref, mag = logprobs_grad64(z[:, -1], tokens, g, h, 1.0, -100)
    within(d, ref, HALF[dtype] * ref.abs() + 2.0 ** -24 * 200 * mag + TINY[dtype])


def test_kept_statistics_of_other_rows_are_refused():
    z, tokens, g = torch.randn(4, 30, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones(4, device="cuda")
    keep = {}
    raw.token_log_probs(z[:3], tokens[:3], keep=keep)
    for bad in (keep, {"stats": None, "entropy": g}, {"stats": torch.zeros(4, 2), "entropy": g}, {"stats": torch.zeros(4, 2, device="cuda"), "entropy": g.double()}):
        with pytest.raises(ValueError):
            raw.token_log_probs_grad(z, tokens, bad, g, None)


def test_two_streams_at_once():
    """Calls on two streams side by side, each of which has workspaces of its own, give what each gives alone."""
    ids = [ids_for(3000, 500, "zipf", s).cuda() for s in (1, 2)]
    dy = torch.randn(3000, 136, device="cuda", dtype=torch.bfloat16)
    z = [torch.randn(40, 20001, device="cuda") for _ in range(2)]
    tokens = torch.arange(40, device="cuda")

    def work(i):
        return [raw.embedding_grad(ids[i], dy, 500), *raw.token_log_probs(z[i], tokens, 8)]

    alone = [work(0), work(1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, alone[i]))


@pytest.mark.parametrize("rows,vocab", [(1190, 4099), (1190, 40001), (3000, 2100), (2961, 4100), (100, 5000), (150, 17000)])
def test_rows_of_every_length_agree(rows, vocab):
    """Few and many rows are worked on by CTAs of different sizes: the same row gives the same alternatives, and the numbers up to the order
    of its sums."""
    z = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)) * 3).to(torch.bfloat16)
    z[1], z[2, : vocab // 2], z[3] = -math.inf, -math.inf, 1.0
    z[4, 7] = z[4, vocab - 1] = 60.0
    tokens = torch.arange(rows) % vocab
    many = raw.token_log_probs(z.cuda(), tokens.cuda(), 9)
    some = torch.cat([torch.arange(8), torch.arange(rows - 3, rows)])
    lp, ent, tv, ti, *_ = logprobs64(z[some], tokens[some], 9, 1.0, -100)
    assert torch.equal(many.top_indices.cpu()[some], ti)
    tol_lp, tol_ent = _tolerances(z[some], tokens[some], lp, ent, vocab, 1.0)
    within(many.log_probs[some.cuda()], lp, tol_lp)
    within(many.entropy[some.cuda()], ent, tol_ent)


def test_offsets_beyond_32_bits():
    far = 2 ** 31 + 16  # elements between two rows
    space = torch.empty(far + 1024, dtype=torch.bfloat16, device="cuda")
    rows = space.as_strided((2, 1000), (far, 1))
    rows.copy_(torch.randn(2, 1000))
    near = rows.contiguous()
    ids = torch.tensor([1, 0, 1], device="cuda")
    assert torch.equal(raw.embedding_lookup(ids, rows, 2.0), raw.embedding_lookup(ids, near, 2.0))
    one = torch.tensor([0, 1], device="cuda")
    assert torch.equal(raw.embedding_grad(one, rows, 3), raw.embedding_grad(one, near, 3))
    kept, plain = {}, {}
    a, b = raw.token_log_probs(rows, one, 4, keep=kept), raw.token_log_probs(near, one, 4, keep=plain)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    g = torch.randn(2, device="cuda")
    assert torch.equal(raw.token_log_probs_grad(rows, one, kept, g, g), raw.token_log_probs_grad(near, one, plain, g, g))


@pytest.mark.parametrize("n", [100, 600])
def test_embedding_gradient_into_the_memory_of_its_input(n):
    ids = ids_for(n, n, "zipf", 5).cuda()
    dy = torch.randn(n, 64, device="cuda")
    ref = raw.embedding_grad(ids, dy, n, 0.5)
    space = torch.empty(2 * n, 64, device="cuda")
    for at in (0, 1, n // 2):  # the same rows, and rows some of which are the other's
        inner = space[at:at + n]
        inner.copy_(dy)
        assert torch.equal(raw.embedding_grad(ids, inner, n, 0.5, out=space[:n]), ref)
    space[:n] = dy
    assert torch.allclose(raw.embedding_grad(ids, space[:n], n, 0.5, out=space[:n], accumulate=True), ref + dy, atol=1e-6)


def test_ids_that_no_tensor_holds():
    from tests.test_vocab_cpu import IDS_OF_NOTHING, test_ids_that_no_tensor_holds as check

    for value in IDS_OF_NOTHING:
        check(value, "cuda")
