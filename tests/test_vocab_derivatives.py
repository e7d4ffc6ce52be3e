"""Derivatives of the embedding and of token log probabilities other than the ordinary backward pass: carried or refused, never dropped."""
import pytest
import torch
from torch.autograd import forward_ad

from tnn_b200.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _calls(device):
    gen = torch.Generator().manual_seed(1)
    ids = torch.tensor([3, 0, 3, 5, 1, 2], device=device)
    table, logits = torch.randn(7, 8, generator=gen).to(device), torch.randn(6, 40, generator=gen).to(device)
    return [(table, lambda t: F.embedding(ids, t, 0.5)), (logits, lambda t: F.token_log_probs(t, ids).log_probs),
            (logits, lambda t: F.token_log_probs(t, ids, 2).entropy)]


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_on_the_cpu(which, no_grad):
    x, call = _calls("cpu")[which]
    v = torch.randn(x.shape, generator=torch.Generator().manual_seed(2))
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        tangent = forward_ad.unpack_dual(call(forward_ad.make_dual(x, v))).tangent
    x64, v64 = x.double(), v.double()
    difference = (call(x64 + 1e-5 * v64) - call(x64 - 1e-5 * v64)) / 2e-5  # off by 1e-10 times a third derivative, 1e-16 / 1e-5 of rounding
    assert torch.allclose(tangent.double(), difference, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused_on_the_gpu(which, no_grad):
    x, call = _calls("cuda")[which]
    alone = call(x)
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        with pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        assert torch.equal(call(x), alone)  # tensors without a tangent are not affected


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
def test_transforms_are_refused_on_the_gpu(which):
    x, call = _calls("cuda")[which]
    for transform in (lambda: torch.func.jvp(call, (x,), (torch.ones_like(x),)), lambda: torch.func.grad(lambda t: call(t).sum())(x),
                      lambda: torch.func.vmap(call)(torch.stack([x, x]))):
        with pytest.raises(RuntimeError):
            transform()


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
def test_gradients_that_carry_more_than_numbers_are_refused_on_the_gpu(which):
    x, call = _calls("cuda")[which]
    x.requires_grad_()
    y = call(x)
    one = torch.ones_like(y)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, torch.stack([one, one]), is_grads_batched=True, retain_graph=True)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, x, forward_ad.make_dual(one, one), retain_graph=True)
        inside, = torch.autograd.grad(y, x, one, retain_graph=True)
    outside, = torch.autograd.grad(y, x, one)
    assert torch.equal(inside, outside)
