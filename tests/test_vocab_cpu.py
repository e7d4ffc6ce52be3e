"""Token embedding with scaling and token log probabilities on CPU tensors: definitions, gradients against differences, refusals."""
import math

import pytest
import torch

from tests._vocab_reference import embedding64, embedding_grad64, ids_for, logits_for, logprobs64, logprobs_grad64
from tnn_b200.ops import functional as F
from tnn_b200.ops import raw

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("padding", [None, 3])
def test_embedding_and_its_gradient(dtype, padding):
    ids = ids_for(57, 23, "zipf", 1).view(3, 19)
    ids[0, 0], ids[2, 2] = 40, -3  # outside of the table: row 0
    table = torch.randn(23, 13).to(dtype)
    y = raw.embedding_lookup(ids, table, 1.7, padding)
    assert y.shape == (3, 19, 13) and y.dtype == dtype
    ref = embedding64(ids.view(-1), table, 1.7, padding)
    # one rounding of the product in fp32, one to the type
    assert bool(((y.view(57, 13).double() - ref).abs() <= (HALF[dtype] + 2 ** -23) * ref.abs() + 1e-30 + (6e-8 if dtype == torch.float16 else 0)).all())
    dy = torch.randn(3, 19, 13).to(dtype)
    d = raw.embedding_grad(ids, dy, 23, 1.7, padding)
    ref, mag, count = embedding_grad64(ids.view(-1), dy.view(57, 13), 23, 1.7, padding)
    tol = HALF[dtype] * ref.abs() + (count[:, None] + 2) * 2 ** -24 * mag * (1 + HALF[dtype]) + (6e-8 if dtype == torch.float16 else 0)
    assert d.dtype == dtype and bool(((d.double() - ref).abs() <= tol + 1e-30).all())
    out = torch.ones(23, 13)
    assert raw.embedding_grad(ids, dy, 23, 1.7, padding, out, accumulate=True) is out
    assert torch.allclose(out.double(), ref + 1, atol=1e-5)


def test_embedding_autograd():
    ids = ids_for(31, 9, "zipf", 2)
    table = torch.randn(9, 5, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda w: F.embedding(ids, w, 0.3, 2), (table,))
    y = F.embedding(ids, table, 2.0)
    y.sum().backward()  # a gradient of stride 0
    assert torch.equal(table.grad, 2.0 * torch.bincount(ids, minlength=9).double()[:, None].expand(9, 5))


KINDS = ["plain", "masked", "few", "equal", "coarse", "rising", "peaked", "bad"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("top", [0, 1, 7])
def test_token_log_probs(kind, top):
    z = logits_for(9, 31, torch.float32, kind, 3)
    tokens = torch.randint(0, 31, (9,), generator=torch.Generator().manual_seed(4))
    tokens[1], tokens[3] = -100, 31
    r = raw.token_log_probs(z.view(3, 3, 31), tokens.view(3, 3), top, 0.7)
    lp, ent, tv, ti, *_ = logprobs64(z, tokens, top, 0.7, -100)
    assert r.log_probs.shape == (3, 3) and r.top_indices.shape == (3, 3, top)
    assert torch.equal(r.top_indices.view(9, top), ti)
    for got, ref in ((r.log_probs.view(9), lp), (r.entropy.view(9), ent), (r.top_log_probs.view(9, top), tv)):
        assert torch.allclose(got.double(), ref, rtol=1e-5, atol=1e-5, equal_nan=True)


def test_token_log_probs_autograd():
    z = logits_for(6, 11, torch.float64, "plain", 5).requires_grad_()
    tokens = torch.tensor([0, 3, -100, 10, 5, 5])

    def both(z):
        r = F.token_log_probs(z, tokens, 3, 0.8)
        return r.log_probs, r.entropy

    assert torch.autograd.gradcheck(both, (z,))
    r = F.token_log_probs(z, tokens, 3, 0.8)
    assert not r.top_log_probs.requires_grad and not r.top_indices.requires_grad
    g, h = torch.randn(6, dtype=torch.float64), torch.randn(6, dtype=torch.float64)
    d = torch.autograd.grad((r.log_probs, r.entropy), (z,), (g, h))[0]
    assert torch.allclose(d, logprobs_grad64(z.detach(), tokens, g, h, 0.8, -100)[0])
    only = torch.autograd.grad(F.token_log_probs(z, tokens).entropy.sum(), z)[0]
    assert torch.allclose(only, logprobs_grad64(z.detach(), tokens, torch.zeros(6), torch.ones(6), 1.0, -100)[0])


def test_rows_without_a_distribution_get_no_gradient():
    z = logits_for(8, 17, torch.float32, "masked", 6).requires_grad_()
    r = F.token_log_probs(z, torch.arange(8), 2)
    (r.log_probs.clamp_min(-1e4).sum() + r.entropy.sum()).backward()
    assert torch.equal(z.grad[4], torch.zeros(17)) and r.log_probs[4].item() == -math.inf and r.entropy[4].item() == 0
    assert bool(torch.isfinite(z.grad).all())


def _refusals(dev):
    ids, table = torch.zeros(4, dtype=torch.int64, device=dev), torch.zeros(5, 8, device=dev)
    z, dy = torch.zeros(4, 9, device=dev), torch.zeros(4, 8, device=dev)
    return [
        (TypeError, lambda: raw.embedding_lookup(ids.float(), table)),
        (ValueError, lambda: raw.embedding_lookup(ids, table[0])),
        (ValueError, lambda: raw.embedding_lookup(ids, table.long())),
        (ValueError, lambda: raw.embedding_lookup(ids, table[:0])),
        (TypeError, lambda: raw.embedding_grad(ids.short(), dy, 5)),
        (ValueError, lambda: raw.embedding_grad(ids[:3], dy, 5)),
        (ValueError, lambda: raw.embedding_grad(ids, dy, 0)),
        (ValueError, lambda: raw.embedding_grad(ids, dy, 5, accumulate=True)),
        (ValueError, lambda: raw.embedding_grad(ids, dy, 5, out=torch.zeros(4, 8, device=dev))),
        (ValueError, lambda: raw.embedding_grad(ids, dy, 5, out=torch.zeros(8, 5, device=dev).t())),
        (TypeError, lambda: raw.embedding_grad(ids, dy.half(), 5, out=torch.zeros(5, 8, device=dev, dtype=torch.bfloat16))),
        (TypeError, lambda: raw.embedding_grad(ids, dy.half(), 5, out=torch.zeros(5, 8, device=dev, dtype=torch.half), accumulate=True)),
        (ValueError, lambda: raw.token_log_probs(z, ids[:3])),
        (ValueError, lambda: raw.token_log_probs(z.long(), ids)),
        (TypeError, lambda: raw.token_log_probs(z, ids.float())),
        (ValueError, lambda: raw.token_log_probs(z, ids, top_k=10)),
        (ValueError, lambda: raw.token_log_probs(torch.zeros(4, 90, device=dev), ids, top_k=33)),
        (ValueError, lambda: raw.token_log_probs(z, ids, top_k=-1)),
        (ValueError, lambda: raw.token_log_probs(z, ids, temperature=0.0)),
        (ValueError, lambda: raw.token_log_probs(z, ids, temperature=math.nan)),
        (ValueError, lambda: raw.token_log_probs(z[:, :0], ids)),
    ]


@pytest.mark.parametrize("i", range(len(_refusals("cpu"))))
def test_refusals(i):
    error, call = _refusals("cpu")[i]
    with pytest.raises(error):
        call()


def test_empty_batches():
    none = torch.zeros(2, 0, dtype=torch.int64)
    assert raw.embedding_lookup(none, torch.zeros(3, 4)).shape == (2, 0, 4)
    assert torch.equal(raw.embedding_grad(none, torch.zeros(2, 0, 4), 3), torch.zeros(3, 4))
    r = raw.token_log_probs(torch.zeros(2, 0, 5), none, 2)
    assert r.log_probs.shape == (2, 0) and r.top_indices.shape == (2, 0, 2)


@pytest.mark.parametrize("value,T", [(-1e9, 1.0), (-1e9, 0.1), (-1e10, 0.8), (-1e15, 1.0), (1e10, 0.8), (5000.0, 1e-6), (1e34, 1e-6),
                                     (torch.finfo(torch.float32).min, 0.8)])
def test_rows_of_large_logits(value, T):
    """Rows filled with a finite mask value, large logits, small temperatures: the distances to the maximum count, not the size."""
    z = torch.full((3, 1000), value)
    z[1, ::3] = -math.inf
    z[2, 17:19] = value + abs(value) / 2
    tokens, g, h = torch.tensor([0, 1, 18]), torch.tensor([0.5, -1.0, 2.0]) * T, torch.tensor([1.0, 0.7, -0.3]) * T
    lp, ent, tv, ti, *_ = logprobs64(z, tokens, 3, T, -100)
    z.requires_grad_()
    r = F.token_log_probs(z, tokens, 3, T)
    assert torch.equal(r.top_indices, ti)
    # sums of 1000 equal terms, a logarithm below 7 and a product with it: 1000 steps of 2^-24 each and a few more; the distance to the
    # maximum, 5e14 among these, its quotient by the temperature, the result and the reference are rounded to fp32 (or are infinite there)
    for got, ref in ((r.log_probs, lp), (r.entropy, ent), (r.top_log_probs, tv)):
        assert torch.allclose(got.detach().double(), ref.float().double(), rtol=4 * 2.0 ** -24, atol=7 * 1100 * 2.0 ** -24)
    (d,) = torch.autograd.grad((r.log_probs, r.entropy), (z,), (g, h))
    ref, mag = logprobs_grad64(z.detach(), tokens, g, h, T, -100)
    assert bool(((d.double() - ref).abs() <= 8 * 1100 * 2.0 ** -24 * mag + 1e-12).all())


def test_rows_longer_than_32_bit_counts_are_refused():
    """Widths beyond 32 bits were cut off on their way into the kernels."""
    ids, one = torch.zeros(1, dtype=torch.int64), torch.zeros(1, 1)
    for width in (2 ** 30 + 1, 2 ** 31 + 8, 2 ** 32 + 8):
        with pytest.raises(ValueError):
            raw.embedding_lookup(ids, one.expand(1, width))
        with pytest.raises(ValueError):
            raw.embedding_grad(ids, one.expand(1, width), 1)


IDS_OF_NOTHING = [None, 2 ** 64, -2 ** 64 + 3, 2 ** 63, 2 ** 32, 2 ** 31 + 1]


@pytest.mark.parametrize("value", IDS_OF_NOTHING)
def test_ids_that_no_tensor_holds(value, dev="cpu"):
    """A padding index or an ignored token beyond 32 or 64 bits is no id's, whatever its lowest bits are."""
    ids, table = torch.tensor([0, 1, 3, -1], device=dev), torch.randn(5, 8, device=dev)
    z, tokens = torch.randn(4, 9, device=dev), torch.tensor([0, 1, 3, 2], device=dev)
    far = -7 if value is None else value
    for kind in (torch.int64, torch.int32):
        assert torch.equal(raw.embedding_lookup(ids.to(kind), table, 1.0, value), raw.embedding_lookup(ids, table))
        assert torch.equal(raw.embedding_grad(ids.to(kind), table[:4], 5, 1.0, value), raw.embedding_grad(ids, table[:4], 5))
        kept, plain = {}, {}
        for a, b in zip(raw.token_log_probs(z, tokens.to(kind), 2, 1.0, far, kept), raw.token_log_probs(z, tokens, 2, keep=plain)):
            assert torch.equal(a, b)
        assert torch.equal(raw.token_log_probs_grad(z, tokens.to(kind), kept, z[:, 0], z[:, 1], 1.0, far),
                           raw.token_log_probs_grad(z, tokens, plain, z[:, 0], z[:, 1]))


def test_kept_entropies_of_other_rows_are_refused():
    """One row's would be spread over all of them."""
    z, tokens, g, keep = torch.randn(4, 30), torch.zeros(4, dtype=torch.int64), torch.ones(4), {}
    raw.token_log_probs(z[:1], tokens[:1], keep=keep)
    for bad in (keep, {"stats": None, "entropy": torch.zeros(3)}, {"stats": None, "entropy": None}):
        with pytest.raises(ValueError):
            raw.token_log_probs_grad(z, tokens, bad, None, g)
