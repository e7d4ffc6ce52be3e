"""Token log probabilities of rows whose logits, in units of the temperature, are larger than fp32's whole numbers: rows filled with a
finite mask value, large logits, small temperatures."""
import math

import pytest
import torch

from tests._vocab_reference import logprobs64, logprobs_grad64
from tests.test_vocab_gpu import HALF, TINY, _tolerances, within
from tnn_b200.ops import functional as F
from tnn_b200.ops import raw

pytestmark = pytest.mark.gpu
FAR = [(-1e9, 1.0), (-1e9, 0.3), (-1e9, 0.1), (-1e10, 1.0), (-1e10, 0.8), (-1e12, 1.0), (-1e15, 1.0), (-1e30, 0.8), (1e10, 0.8), (1e15, 1.0),
       (5000.0, 1e-6), (-50000.0, 1e-5), (11.0, 1e-6)]
EDGE = 2.0 ** 24 / 1.4426950408889634  # here z log2(e) reaches 2^24


def rows_at(value, vocab, dtype):
    """Every logit the same; a third of them lower; half of them ruled out; one above all others; ordinary numbers around the value."""
    z = torch.full((5, vocab), value)
    z[1, ::3] = value - abs(value) / 2
    z[2, : vocab // 2] = -math.inf
    z[3, vocab // 3] = value + abs(value) / 2
    z[4] += torch.randn(vocab, generator=torch.Generator().manual_seed(vocab)) * 2
    return z.to(dtype)


def check(z, T, top, what):
    rows, vocab = z.shape
    tokens = torch.arange(rows) * 3 % vocab
    lp, ent, tv, ti, _, p, _ = logprobs64(z, tokens, top, T, -100)
    zc = z.cuda().requires_grad_()
    r = F.token_log_probs(zc, tokens.cuda(), top, T)
    assert torch.equal(r.top_indices.cpu(), ti), what
    tol_lp, tol_ent = _tolerances(z, tokens, lp, ent, vocab, T)
    within(r.log_probs.detach(), lp, tol_lp, f"{what}: log probability")
    within(r.entropy.detach(), ent, tol_ent, f"{what}: entropy")
    within(r.top_log_probs, tv, tol_lp.max() + 2.0 ** -22 * torch.where(torch.isfinite(tv), tv, 0.0).abs(), f"{what}: alternatives")
    gen = torch.Generator().manual_seed(rows)
    g, h = torch.randn(rows, generator=gen) * T, torch.randn(rows, generator=gen) * T  # (their quotients by T stay in fp16's range)
    (d,) = torch.autograd.grad((r.log_probs, r.entropy), (zc,), (g.cuda(), h.cuda()))
    ref, mag = logprobs_grad64(z, tokens, g, h, T, -100)
    # a probability is off by the sum's error (chain as in _tolerances) and by a few half steps of its exponent, the distance to the maximum
    # (those beyond 200 are zero); the entropy's error and a few products come on top; probabilities below 2^-126 are flushed
    far = ((z.double().max(1, keepdim=True).values - z.double()) / T).nan_to_num(0, 0, 0).clamp(max=200)
    lost = 2.0 ** -126 * (g.abs() + h.abs() * (88 + math.log(vocab))).double()[:, None] / T
    tol = HALF[z.dtype] * ref.abs() + 2.0 ** -24 * (vocab / 256 + 40 + 8 * far) * mag + p * (h.double().abs() * tol_ent)[:, None] / T + lost
    within(d, ref, tol + TINY[z.dtype], f"{what}: gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 9, 1000, 20003, 131072])
@pytest.mark.parametrize("value,T", FAR)
def test_far_rows(dtype, vocab, value, T):
    if 1.5 * abs(value) > torch.finfo(dtype).max:
        pytest.skip("no number of this type")
    check(rows_at(value, vocab, dtype), T, min(vocab, 6), f"{value} / {T}")


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("order", ["mixed", "rising", "falling"])
@pytest.mark.parametrize("vocab", [40, 5000, 131072])
def test_rows_across_the_edge(sign, order, vocab):
    """The running maximum passes from logits whose product with log2(e) is rounded to those where it is not, within few nats."""
    z = sign * EDGE + torch.randint(-12, 13, (6, vocab), generator=torch.Generator().manual_seed(vocab)).double()
    if order != "mixed":
        z = z.sort(1, descending=order == "falling").values
    check(z.float(), 1.0, 4, f"{order} {sign}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1e-6, 1e-4, 1e4, 1e6])
def test_ordinary_logits_at_extreme_temperatures(dtype, T):
    z = (torch.randn(7, 9001, generator=torch.Generator().manual_seed(3)) * 2.5).to(dtype)
    z[2, 100:104] = z[2].max() + 1  # the maximum four times
    z[3, ::2] = -math.inf
    check(z, T, 5, f"T {T}")


def test_the_edge_is_where_it_is_said_to_be():
    """A row just below the edge and one just above differ by no more than their logits do."""
    for v in (EDGE - 40, EDGE + 40):
        r = raw.token_log_probs(torch.full((1, 77), float(v), device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"))
        assert abs(r.log_probs.item() + math.log(77)) < 1e-5 and abs(r.entropy.item() - math.log(77)) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,weight", [(1e-6, 1e10), (1e-3, 1e16), (0.8, 1e22)])
def test_large_entropy_gradients_leave_ruled_out_tokens_alone(dtype, T, weight):
    z = torch.randn(4, 1003, generator=torch.Generator().manual_seed(5)).to(dtype)
    z[:, 1::2] = -math.inf
    z[1, 1::2] = torch.finfo(dtype).min
    z[2, 40:44:2] = 5.0
    tokens, h = torch.tensor([0, 2, 40, 4], device="cuda"), torch.full((4,), weight, device="cuda")
    keep = {}
    raw.token_log_probs(z.cuda(), tokens, 0, T, keep=keep)
    d = raw.token_log_probs_grad(z.cuda(), tokens, keep, None, h, T)
    assert bool((d[:, 1::2] == 0).all())
