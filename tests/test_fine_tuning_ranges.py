"""The ends of the range of the fine-tuning losses and of Adam's moments in 8 bits, in the tensor operations that run on
the CPU and state what the kernels compute: terms of weight 0 that overflow, answers that cannot be, factors of 0,
blocks of the largest and smallest moments, function transforms."""
import math

import pytest
import torch

from t5x_b200 import losses, optimizers


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


def impossible(row):
  """Two pairs over a vocabulary of 3; the target of one token of `row` has a logit of -inf."""
  x = torch.tensor([[[1.0, 2.0, 0.5], [0.0, -1.0, 3.0]], [[0.3, 0.2, 0.1], [2.0, 2.0, 2.0]],
                    [[0.1, 0.2, 0.9], [0.5, 0.6, 0.1]], [[0.7, 0.1, 0.3], [0.2, 1.0, 0.4]]], dtype=torch.float64)
  t = torch.tensor([[1, 2], [0, 1], [2, 0], [1, 1]])
  x[row, 1, t[row, 1]] = -math.inf
  return x.requires_grad_(), t


@pytest.mark.parametrize("from_scores", [False, True])
def test_preference_of_an_impossible_answer(from_scores):
  """Rejected: margin +inf, log(1 + exp(-inf)) = 0 and no gradient; preferred: margin -inf, an infinite loss."""
  r = torch.zeros(4)

  def call(x, t, **kw):
    if not from_scores:
      return losses.compute_preference_loss(x, t, None, r, **kw)
    logp = x.log_softmax(-1).gather(-1, t[..., None])[..., 0]
    return losses.preference_loss_from_token_scores(logp, None, r, **kw)

  x, t = impossible(1)
  loss, scores, margins, pairs = call(x, t)
  other = losses.compute_preference_loss(x[2:].detach(), t[2:], None, r[2:])[0]
  assert loss.item() == pytest.approx(other.item(), rel=1e-12) and pairs.item() == 2
  assert scores[1].item() == -math.inf and margins[0].item() == math.inf
  grad = torch.autograd.grad(loss, x)[0]
  assert torch.all(grad[:2] == 0) and torch.all(torch.isfinite(grad)) and torch.all(grad[2:] != 0)
  assert call(x, t, label_smoothing=0.1)[0].item() == math.inf
  x, t = impossible(0)
  assert call(x, t)[0].item() == math.inf and call(x, t)[2][0].item() == -math.inf
  assert call(x, t, label_smoothing=1.0)[0].item() < math.inf


def test_normalizing_factor_of_zero():
  """No tokens in the batch: the quotient that tensor operations give, no exception."""
  x, t, one = torch.randn(2, 3, 5), torch.zeros(2, 3, dtype=torch.long), torch.ones(2, 3)
  for factor in (0.0, torch.tensor(0.0)):
    assert losses.compute_preference_loss(x, t, one, torch.zeros(2), loss_normalizing_factor=factor)[0].item() == math.inf
    assert math.isnan(losses.compute_policy_loss(x, t, 0 * one, -one, torch.ones(2),
                                                 loss_normalizing_factor=factor)[0].item())


def test_function_transforms():
  gen = torch.Generator().manual_seed(0)
  x = torch.randn(4, 3, 7, generator=gen, dtype=torch.float64)
  t = torch.randint(0, 7, (4, 3), generator=gen)
  r, old = torch.randn(4, generator=gen), -2 + torch.randn(4, 3, generator=gen)
  for loss in (lambda v: losses.compute_preference_loss(v, t, None, r)[0],
               lambda v: losses.compute_policy_loss(v, t, None, old, r)[0]):
    leaf = x.clone().requires_grad_()
    want = torch.autograd.grad(loss(leaf), leaf)[0]
    assert torch.allclose(torch.func.grad(loss)(x), want, rtol=1e-12, atol=1e-15)


# ---- moments in 8 bits ----
@pytest.mark.parametrize("second", [False, True])
@pytest.mark.parametrize("largest", [1.2e-38, 1e-37, 5e-36, 1e-33, 1e-30, 1.0, 8e37, 9e37, 3.4e38])
def test_moments_at_the_ends_of_the_range(largest, second):
  gen = torch.Generator().manual_seed(1)
  x = torch.rand(600, generator=gen, dtype=torch.float64) ** 4 * (1 if second else -1)
  x[::7] *= 1 if second else -1
  x[::50] = 0
  x[1::256] = 1
  x = (x * largest).float()
  codes, absmax = optimizers.quantize_moment(x, optimizers._moment_noise(600, 3, 9, "cpu") & 0xFFFF, second,
                                             2.0 ** -100)  # (as the step stores them)
  back = optimizers.dequantize_moment(codes, absmax)
  assert torch.all(torch.isfinite(back))
  # one step of e4m3 at most: an eighth of the value, or 2^-9 / 448 of the scale
  step = x.abs().double() / 8 + max(largest, 2.0 ** -100) / (448 * 512) * 1.001
  assert torch.all((back.double() - x.double()).abs() <= step)
  assert torch.all((back > 0) == (x > 0)) if second else torch.all(back.sign() * x.sign() >= 0)
  if second:
    assert float(back[x > 0].min()) >= 2.0 ** -118


def test_zero_gradients_behind_smallest_ones():
  """A second moment of 8e-44 is not zero when no gradient follows: the next steps are bounded by it, not by eps."""
  g = {"w": torch.full((300,), 4e-22)}
  t = optimizers.scale_by_adam8(b2=0.5, eps=1e-30)
  state = t.init(g)
  for i in range(60):
    out, state = t.update(g if i == 0 else {"w": torch.zeros(300)}, state)
    assert float(out["w"].abs().max()) < 100


def test_overflowing_second_moment_shows():
  """A square beyond 32 bits: its block is NaN when it is read back, as behind a NaN, not a step of 0 for good."""
  w = {"w": torch.ones(600)}
  opt = optimizers.adamw8(1e-2, weight_decay=0.0).create(w)
  g = torch.ones(600)
  g[300] = 1e20
  opt = opt.apply_gradient({"w": g})
  assert torch.all(torch.isfinite(opt.target["w"]))
  assert torch.isnan(opt.state.param_states["0"]["nu_absmax"]["w"]).tolist() == [False, True, False]
  opt = opt.apply_gradient({"w": torch.ones(600)})
  assert torch.isnan(opt.target["w"]).nonzero().flatten().tolist() == list(range(256, 512))


# ---- refusals of the C entry points, with made-up addresses: nothing is launched ----
A = 1 << 20


@pytest.mark.parametrize("at,bytes_of", [(0, 16), (1, 8), (2, 4), (3, 4), (4, 4), (5, 4), (6, 4)])
def test_misaligned_pointers_are_refused(at, bytes_of):
  """Scratch, targets and values of 32 bits; with the middle of them an access would fault."""
  from t5x_b200.ops import native
  lib = native.lib()
  p = [A] * 7
  p[at] += bytes_of // 2
  scratch, targets, weights, old, ref, adv, out = p
  calls = [lambda: lib.t5x_policy_loss(A, 1, A, 4, 3, 8, 24, 8, targets, weights, old, ref, adv, 3, 1, 0.2, 0.2, 0.1, 1.0,
                                       None, scratch, out, None),
           lambda: lib.t5x_policy_loss_tokens(A, A, 4, 3, weights, old, ref, adv, 3, 1, 0.2, 0.2, 0.1, 1.0, None, scratch,
                                              out, None),
           lambda: lib.t5x_preference_loss(A, 1, A, 4, 3, 8, 24, 8, targets, weights, ref, 0.1, 0.0, 1.0, old, scratch, adv,
                                           A, out, None),
           lambda: lib.t5x_preference_loss_tokens(A, A, 4, 3, weights, ref, 0.1, 0.0, 1.0, old, scratch, A, adv, out,
                                                  None)]
  for i, call in enumerate(calls):
    if at == 1 and i % 2:
      continue  # (no targets)
    assert call() != 0, i
    assert "misaligned" in lib.t5x_last_error().decode()
  assert lib.t5x_scale_gradient(A + 2, A, 4, 1, A, None) != 0 and lib.t5x_scale_gradient(A, A + 1, 4, 0, A, None) != 0
  assert lib.t5x_scale_gradient(A, A, 4, 1, A + 2, None) != 0
