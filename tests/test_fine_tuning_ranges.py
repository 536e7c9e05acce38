"""The ends of the range of the fine-tuning losses and of Adam's moments in 8 bits, in the tensor operations that run on
the CPU and state what the kernels compute: terms of weight 0 that overflow, answers that cannot be, factors of 0,
blocks of the largest and smallest moments, function transforms."""
import math

import pytest
import torch

from t5x_b200 import losses


@pytest.mark.parametrize("kl_weight", [0.0, 0.1])
def test_policy_reference_far_above(kl_weight):
  """exp(ref - logp) overflows 32 bits: with weight 0 (the default) the term is not part of the loss."""
  logits = torch.tensor([[[0.0, 100.0]]], requires_grad=True)
  loss, kl, clipped, weight = losses.compute_policy_loss(
      logits, torch.tensor([[0]]), None, torch.tensor([[-100.0]]), torch.tensor([1.0]), torch.tensor([[-1.0]]),
      kl_weight=kl_weight)
  assert kl.item() == math.inf and clipped.item() == 0 and weight.item() == 1
  if kl_weight:
    assert loss.item() == math.inf
    return
  # logp = -100 and ratio 1 to 2^-24 * 100 each; softmax (e^-100, 1)
  assert loss.item() == pytest.approx(-1.0, abs=2e-5)
  assert torch.autograd.grad(loss, logits)[0].flatten().tolist() == pytest.approx([-1.0, 1.0], abs=2e-5)


def test_policy_of_an_impossible_token():
  """A token that the model now rules out: ratio 0, and a KL term of infinity where it is asked for."""
  x = torch.tensor([[[0.0, -math.inf, 0.5]]], requires_grad=True)
  one = torch.ones(1, 1)
  call = lambda w: losses.compute_policy_loss(x, torch.tensor([[1]]), None, -one, one[0], -2 * one, kl_weight=w)  # noqa: E731
  out = call(0.0)
  assert out[0].item() == 0 and out[1].item() == math.inf and call(0.1)[0].item() == math.inf
  assert torch.all(torch.autograd.grad(out[0], x)[0] == 0)
