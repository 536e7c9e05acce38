"""Losses of preference and policy fine-tuning as tensor operations (what runs on the CPU and states what the kernels
compute): against hand-computed values, gradients against differences, masked places, refusals."""
import math

import pytest
import torch

from t5x_b200 import losses


def log_softmax_at(x, t):
  m = max(x)
  return x[t] - m - math.log(sum(math.exp(v - m) for v in x))


def test_preference_by_hand():
  x = [[[1.0, 2.0, 0.5], [0.0, -1.0, 3.0]], [[0.3, 0.2, 0.1], [2.0, 2.0, 2.0]]]
  t, w, r = [[1, 2], [0, 1]], [[1.0, 0.5], [1.0, 0.0]], [-0.7, -1.3]
  s = [sum(w[b][i] * log_softmax_at(x[b][i], t[b][i]) for i in range(2)) for b in range(2)]
  d = 0.3 * ((s[0] - r[0]) - (s[1] - r[1]))
  want = (0.9 * math.log(1 + math.exp(-d)) + 0.1 * math.log(1 + math.exp(d))) / 4
  loss, scores, margins, pairs = losses.compute_preference_loss(
      torch.tensor(x, dtype=torch.float64), torch.tensor(t), torch.tensor(w), torch.tensor(r), beta=0.3,
      label_smoothing=0.1, loss_normalizing_factor=4)
  assert loss.item() == pytest.approx(want, rel=1e-6) and scores.tolist() == pytest.approx(s, rel=1e-12)
  assert margins.item() == pytest.approx(d, rel=1e-6) and pairs.item() == 1


@pytest.mark.parametrize("a,old,held", [(1.0, -3.0, True), (1.0, -0.4, False), (-2.0, -3.0, False), (-2.0, -0.1, True),
                                        (0.0, -0.9, False)])
def test_policy_by_hand(a, old, held):
  x, ref = [0.5, 1.5, -1.0], -0.8
  logp = log_softmax_at(x, 1)
  ratio = math.exp(logp - old)
  each = -min(a * ratio, a * min(max(ratio, 0.8), 1.3))
  kl = math.exp(ref - logp) - 1 - (ref - logp)
  logits = torch.tensor([[x]], dtype=torch.float64, requires_grad=True)
  loss, k, clipped, weight = losses.compute_policy_loss(
      logits, torch.tensor([[1]]), torch.tensor([[0.5]]), torch.tensor([[old]], dtype=torch.float64),
      torch.tensor([a]), torch.tensor([[ref]], dtype=torch.float64), clip_range=0.2, clip_range_high=0.3,
      kl_weight=0.25, loss_normalizing_factor=torch.tensor(2.0))
  assert loss.item() == pytest.approx(0.25 * (each + 0.25 * kl), rel=1e-9, abs=1e-12)
  assert k.item() == pytest.approx(0.25 * kl, rel=1e-9) and weight.item() == 0.5
  assert clipped.item() == (0.5 if held else 0.0)
  by = 0.25 * ((0.0 if held else -a * ratio) + 0.25 * (1 - math.exp(ref - logp)))
  p = [math.exp(log_softmax_at(x, i)) for i in range(3)]
  want = [by * ((i == 1) - p[i]) for i in range(3)]
  assert torch.autograd.grad(loss, logits)[0].flatten().tolist() == pytest.approx(want, rel=1e-9, abs=1e-15)


def inputs(batch, length, vocab, seed=0):
  gen = torch.Generator().manual_seed(seed)
  rand = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
  weights = (torch.rand(batch, length, generator=gen) > 0.3).double() * torch.rand(batch, length, generator=gen)
  return (rand(batch, length, vocab), torch.randint(0, vocab, (batch, length), generator=gen), weights, rand(batch),
          -2 + rand(batch, length), rand(batch, length), -2 + rand(batch, length))


def test_gradients_against_differences():
  x, t, w, r, old, adv, ref = inputs(4, 3, 6)
  x.requires_grad_()
  assert torch.autograd.gradcheck(
      lambda v: losses.compute_preference_loss(v, t, w, r, label_smoothing=0.1, loss_normalizing_factor=3.0)[0], x)
  assert torch.autograd.gradcheck(
      lambda v: losses.compute_policy_loss(v, t, w, old, adv, ref, kl_weight=0.3)[0], x)
  logp = torch.randn(4, 3, dtype=torch.float64, requires_grad=True)
  assert torch.autograd.gradcheck(lambda v: losses.preference_loss_from_token_scores(v, w, r)[0], logp)
  assert torch.autograd.gradcheck(
      lambda v: losses.policy_loss_from_token_scores(v, w, old, adv[:, 0], ref, kl_weight=0.3)[0], logp)


def test_from_logits_is_from_token_scores():
  x, t, w, r, old, adv, ref = inputs(6, 4, 9)
  logp = x.log_softmax(-1).gather(-1, t[..., None])[..., 0]
  for a, b in ((losses.compute_preference_loss(x, t, w, r), losses.preference_loss_from_token_scores(logp, w, r)),
               (losses.compute_policy_loss(x, t, w, old, adv, ref, kl_weight=0.1),
                losses.policy_loss_from_token_scores(logp, w, old, adv, ref, kl_weight=0.1))):
    for u, v in zip(a, b):
      torch.testing.assert_close(u, v, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_places_hold_anything(bad):
  x, t, w, r, old, adv, ref = inputs(4, 5, 6)
  w[0] = 0
  w[1] = 0  # the first pair is padding
  w[2, 3] = 0
  clean = [v.clone() for v in (x, t, r, old, adv, ref)]
  seen = w != 0
  x[~seen] = bad
  t = torch.where(seen, t, torch.full_like(t, -7))
  r[:2], old[~seen], adv[~seen], ref[~seen] = bad, bad, bad, bad
  for leaf, targets, rr, oo, aa, ff in ((x, t, r, old, adv, ref), clean):
    leaf.requires_grad_()
    a = losses.compute_preference_loss(leaf, targets, w, rr)
    b = losses.compute_policy_loss(leaf, targets, w, oo, aa, ff, kl_weight=0.2)
    leaf.out = [v.detach() for v in (*a, *b)] + [torch.autograd.grad(v, leaf)[0] for v in (a[0], b[0])]
  for u, v in zip(x.out, clean[0].out):
    assert torch.equal(u, v) and torch.all(torch.isfinite(u))
  assert x.out[3].item() == 1 and x.out[2][0] == 0 and torch.all(x.out[-1][~seen] == 0)


def test_no_weights_is_all_ones():
  x, t, _, r, old, adv, _ = inputs(4, 5, 6)
  one = torch.ones(4, 5)
  for a, b in zip(losses.compute_preference_loss(x, t, None, r), losses.compute_preference_loss(x, t, one, r)):
    assert torch.equal(a, b)
  for a, b in zip(losses.compute_policy_loss(x, t, None, old, adv), losses.compute_policy_loss(x, t, one, old, adv)):
    assert torch.equal(a, b)


def test_refusals():
  x, t, w, r, old, adv, ref = inputs(4, 5, 6)
  pref, pol = losses.compute_preference_loss, losses.compute_policy_loss
  for call, message in [
      (lambda: pref(x[0], t, w, r), "3 dimensions"), (lambda: pref(x[:3], t[:3], w[:3], r[:3]), "pairs"),
      (lambda: pref(x, t[:, :2], w, r), "targets"), (lambda: pref(x, t, w[:2], r), "weights"),
      (lambda: pref(x, t, w, r[:2]), "reference_scores"), (lambda: pref(x, t.double(), w, r), "whole numbers"),
      (lambda: pref(x.long(), t, w, r), "floating"), (lambda: pref(x, t, w, r, label_smoothing=1.5), "label_smoothing"),
      (lambda: pref(x, t, w, r, beta=math.inf), "beta"),
      (lambda: pref(x, t, w, r, loss_normalizing_factor="NUM_REAL_TARGET_TOKENS"), "special"),
      (lambda: pref(x[:0], t[:0], w[:0], r[:0]), "pairs"),
      (lambda: pol(x, t, w, old[:, :1], adv), "old_token_scores"), (lambda: pol(x, t, w, old, adv[:2]), "advantages"),
      (lambda: pol(x, t, w, old, adv, ref[:1]), "reference_token_scores"),
      (lambda: pol(x, t, w, old, adv, clip_range=1.5), "clip_range"),
      (lambda: pol(x, t, w, old, adv, clip_range_high=-0.1), "clip_range"),
      (lambda: losses.policy_loss_from_token_scores(x, w, old, adv), "2 dimensions"),
      (lambda: losses.preference_loss_from_token_scores(old[:1], w[:1], r[:1]), "pairs")]:
    with pytest.raises(ValueError, match=message):
      call()


# ---- refusals of the C entry points, with made-up addresses: nothing is launched ----
A = 1 << 20


def _policy(lib, logits=A, fp32=1, grad=A, b=4, l=3, v=8, sb=24, st=8, targets=A, w=A, old=A, ref=A, adv=A, scratch=A,
            out=A):
  return lib.t5x_policy_loss(logits, fp32, grad, b, l, v, sb, st, targets, w, old, ref, adv, 3, 1, 0.2, 0.2, 0.1, 1.0,
                             None, scratch, out, None)


def _preference(lib, logits=A, fp32=1, grad=A, b=4, l=3, v=8, sb=24, st=8, targets=A, w=A, ref=A, scratch=A, scores=A,
                margins=A, out=A):
  return lib.t5x_preference_loss(logits, fp32, grad, b, l, v, sb, st, targets, w, ref, 0.1, 0.0, 1.0, None, scratch,
                                 scores, margins, out, None)


@pytest.mark.parametrize("call", [_policy, _preference])
@pytest.mark.parametrize("bad,message", [
    (dict(logits=0), "null"), (dict(targets=0), "null"), (dict(scratch=0), "null"), (dict(out=0), "null"),
    (dict(logits=A + 2, grad=A + 2), "misaligned"), (dict(grad=A + 4), "same place"), (dict(st=7), "overlap"),
    (dict(sb=23), "overlap"), (dict(b=-2), "sizes"), (dict(l=-1), "sizes"), (dict(v=0), "sizes"),
    (dict(fp32=0, logits=A + 1, grad=A + 1), "misaligned")])
def test_entry_refusals(call, bad, message):
  from t5x_b200.ops import native
  lib = native.lib()
  assert call(lib, **bad) != 0
  assert message in lib.t5x_last_error().decode()


def test_other_entry_refusals():
  from t5x_b200.ops import native
  lib = native.lib()
  assert _preference(lib, b=3) != 0 and "pairs" in lib.t5x_last_error().decode()
  assert _preference(lib, b=0) != 0 and "pairs" in lib.t5x_last_error().decode()
  assert _policy(lib, old=0) != 0 and _policy(lib, adv=0) != 0
  assert lib.t5x_scale_gradient(A, None, 4, 1, A, None) != 0
  assert lib.t5x_preference_loss_tokens(A, A, 3, 4, A, A, 0.1, 0.0, 1.0, None, A, A, A, A, None) != 0
  assert lib.t5x_policy_loss_tokens(None, A, 3, 4, A, A, A, A, 4, 1, 0.2, 0.2, 0.1, 1.0, None, A, A, None) != 0
  with pytest.raises(native.NativeError, match="types and shapes"):
    x = torch.zeros(2, 3, 4)
    native.preference_loss(x, None, torch.zeros(2, 2, dtype=torch.long), None, torch.zeros(2), 0.1, 0.0, 1.0, None)
