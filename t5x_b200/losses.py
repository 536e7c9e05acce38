"""Loss functions (API of t5x/losses.py): z-loss cross-entropy and loss normalisation."""
from __future__ import annotations

import enum
import math
from typing import Mapping, Optional, Tuple, Union

import numpy as np
import torch

from t5x_b200.ops import reference as ref


class _CrossEntropyWithLogits(torch.autograd.Function):
  """CE with z-loss and the reference's hand-written gradient (t5x/losses.py:62-124):
  d logits = g * ((1 + 2 z log_z) softmax - targets); the z-loss output carries no gradient."""

  @staticmethod
  def forward(ctx, logits, targets, z_loss):
    logits = logits.float()
    max_logit = logits.max(dim=-1, keepdim=True).values
    shifted = logits - max_logit
    exp_shifted = torch.exp(shifted)
    sum_exp = exp_shifted.sum(dim=-1, keepdim=True)
    log_softmax = shifted - torch.log(sum_exp)
    loss = -(targets * log_softmax).sum(dim=-1)
    log_z = (torch.log(sum_exp) + max_logit).squeeze(-1)
    total_z_loss = z_loss * log_z * log_z
    loss = loss + total_z_loss
    ctx.save_for_backward(targets, exp_shifted, sum_exp, log_z)
    ctx.z_loss = z_loss
    ctx.mark_non_differentiable(total_z_loss)
    return loss, total_z_loss

  @staticmethod
  def backward(ctx, g, _gz):
    targets, exp_shifted, sum_exp, log_z = ctx.saved_tensors
    deriv = (1 + 2 * ctx.z_loss * log_z)[..., None] * exp_shifted / sum_exp - targets
    g_logits = g[..., None] * deriv
    g_targets = -g[..., None] * (torch.log(exp_shifted / sum_exp))
    return g_logits, (g_targets if ctx.needs_input_grad[1] else None), None


def cross_entropy_with_logits(logits: torch.Tensor, targets: torch.Tensor,
                              z_loss: float) -> Tuple[torch.Tensor, torch.Tensor]:
  """logits, soft targets [..., classes] -> (loss incl. z-loss, z-loss), both [...]."""
  return _CrossEntropyWithLogits.apply(logits, targets, float(z_loss))


def compute_weighted_cross_entropy(
    logits: torch.Tensor, targets: torch.Tensor, weights: Optional[torch.Tensor] = None,
    label_smoothing: float = 0.0, z_loss: float = 0.0,
    loss_normalizing_factor: Optional[float] = None):
  """Sum (not mean) of weighted token losses; returns (loss, z_loss, weight_sum)
  (t5x/losses.py:132-193)."""
  if logits.dim() != targets.dim() + 1:
    raise ValueError(f"Incorrect shapes. Got shape {tuple(logits.shape)} logits and "
                     f"{tuple(targets.shape)} targets")
  vocab_size = logits.shape[-1]
  confidence = 1.0 - label_smoothing
  low_confidence = (1.0 - confidence) if vocab_size == 1 else (1.0 - confidence) / (vocab_size - 1)
  normalizing_constant = -(confidence * math.log(confidence) +
                           (vocab_size - 1) * low_confidence * math.log(low_confidence + 1e-20))
  soft_targets = torch.full(logits.shape, low_confidence, dtype=torch.float32,
                            device=logits.device)
  soft_targets.scatter_(-1, targets[..., None].long(), confidence)
  total_loss, total_z_loss = cross_entropy_with_logits(logits, soft_targets, z_loss)
  total_loss = total_loss - normalizing_constant
  return weight_and_normalize(total_loss, total_z_loss, targets, weights,
                              loss_normalizing_factor)


def weight_and_normalize(token_loss, token_z_loss, targets, weights, loss_normalizing_factor):
  """The weighting / normalising tail of `compute_weighted_cross_entropy`."""
  weight_sum = float(np.prod(targets.shape))
  if weights is not None:
    token_loss = token_loss * weights
    token_z_loss = token_z_loss * weights
    weight_sum = weights.sum()
  if loss_normalizing_factor is not None:
    token_loss = token_loss / loss_normalizing_factor
    token_z_loss = token_z_loss / loss_normalizing_factor
  return token_loss.sum(), token_z_loss.sum(), weight_sum


@enum.unique
class SpecialLossNormalizingFactor(enum.Enum):
  """Normalising factors computed from the batch (t5x/losses.py:196-217)."""
  NUM_REAL_TARGET_TOKENS = 1
  NUM_TOTAL_TARGET_TOKENS = 2
  AVERAGE_PER_SEQUENCE = 3


def convert_special_loss_normalizing_factor_to_enum(x: str) -> SpecialLossNormalizingFactor:
  try:
    return SpecialLossNormalizingFactor[x.upper()]
  except KeyError:
    raise ValueError(f'Could not convert string "{x}" to SpecialLossNormalizingFactor')


def _sum_weights_per_segment(positions, segment_ids, weights):
  """For packed rows: per-token total weight of the token's own segment
  (t5x/losses.py:246-275). Inputs [batch, length]."""
  out = torch.zeros_like(weights, dtype=torch.float32)
  b, l = weights.shape
  # segment ids are small positive ints (0 = padding); accumulate per (row, segment).
  seg = segment_ids.long()
  nseg = int(seg.max().item()) + 1 if seg.numel() else 1
  totals = torch.zeros((b, nseg), dtype=torch.float32, device=weights.device)
  totals.scatter_add_(1, seg, weights.float())
  out = totals.gather(1, seg)
  return torch.where(seg != 0, out, torch.zeros_like(out))


def get_loss_normalizing_factor_and_weights(
    loss_normalizing_factor: Optional[Union[float, int, str, SpecialLossNormalizingFactor]],
    batch: Mapping[str, torch.Tensor]):
  """Resolves a special factor into (float-like factor, per-token weights)
  (t5x/losses.py:278-356)."""
  loss_weights = batch.get("decoder_loss_weights", None)
  if loss_normalizing_factor is None or not isinstance(
      loss_normalizing_factor, (str, SpecialLossNormalizingFactor)):
    return loss_normalizing_factor, loss_weights
  if isinstance(loss_normalizing_factor, str):
    loss_normalizing_factor = convert_special_loss_normalizing_factor_to_enum(
        loss_normalizing_factor)
  if loss_weights is None:
    loss_weights = (batch["decoder_target_tokens"] > 0).float()
  if loss_normalizing_factor == SpecialLossNormalizingFactor.NUM_REAL_TARGET_TOKENS:
    output = loss_weights.sum()
  elif loss_normalizing_factor == SpecialLossNormalizingFactor.NUM_TOTAL_TARGET_TOKENS:
    output = float(np.prod(batch["decoder_target_tokens"].shape))
  elif loss_normalizing_factor == SpecialLossNormalizingFactor.AVERAGE_PER_SEQUENCE:
    if "decoder_segment_ids" in batch:
      norm_vec = _sum_weights_per_segment(batch["decoder_positions"],
                                          batch["decoder_segment_ids"], loss_weights)
    else:
      norm_vec = loss_weights.sum(dim=-1, keepdim=True)
    loss_weights = torch.nan_to_num(loss_weights / norm_vec, nan=0.0, posinf=0.0, neginf=0.0)
    output = loss_weights.sum()
  else:
    raise ValueError(f"Unsupported value of loss_normalizing_factor: {loss_normalizing_factor}")
  return _sum_over_data_replicas(output), loss_weights


def _sum_over_data_replicas(factor):
  """A factor derived from the batch counts the GLOBAL batch: the reference evaluates it
  inside the partitioned step over all replicas' examples (t5x/losses.py:278-356 under
  t5x/trainer.py:745-852), and gradients are summed over replicas afterwards. Each rank sees
  only its shard here, so the per-shard counts are added over the data (and expert) axis."""
  import torch.distributed as dist
  from t5x_b200.parallel import state as pstate
  st = pstate.get()
  if st.data_size * st.expert_size <= 1 or st.data_group is None or not dist.is_initialized():
    return factor
  t = torch.as_tensor(factor, dtype=torch.float32, device=st.device).detach().clone().reshape(1)
  dist.all_reduce(t, group=st.data_group)
  return t[0]


# ----------------------------------------------------------------------------
# Preference and policy fine-tuning
# ----------------------------------------------------------------------------
def _check_tokens(what: str, values: torch.Tensor, dims: int, **tokens) -> None:
  if values.dim() != dims:
    raise ValueError(f"{what}: expected a tensor of {dims} dimensions, got shape {tuple(values.shape)}")
  if not values.is_floating_point():
    raise ValueError(f"{what}: expected floating-point values, got {values.dtype}")
  shape, device = values.shape[:2], values.device
  for name, t in tokens.items():
    if t is None:
      continue
    if t.shape != shape:
      raise ValueError(f"{what}: Incorrect shapes. Got shape {tuple(t.shape)} {name} for [batch, length] = "
                       f"{tuple(shape)}")
    if t.device != device:
      raise ValueError(f"{what}: {name} are on {t.device}, the values on {device}")
    if name == "targets" and (t.is_floating_point() or t.dtype == torch.bool):
      raise ValueError(f"{what}: targets must be whole numbers, got {t.dtype}")


def _check_factor(what: str, factor) -> None:
  if isinstance(factor, (str, SpecialLossNormalizingFactor)):
    raise ValueError(f"{what}: resolve a special loss_normalizing_factor with "
                     "get_loss_normalizing_factor_and_weights first")


def _check_preference(what, values, reference_scores, beta, label_smoothing, factor):
  if values.shape[0] % 2 or values.shape[0] == 0:
    raise ValueError(f"{what}: the batch must hold pairs of rows, got {values.shape[0]} rows")
  if reference_scores.shape != values.shape[:1] or reference_scores.device != values.device:
    raise ValueError(f"{what}: reference_scores must be [{values.shape[0]}] on {values.device}, got "
                     f"{tuple(reference_scores.shape)} on {reference_scores.device}")
  if not 0.0 <= label_smoothing <= 1.0 or not math.isfinite(beta):
    raise ValueError(f"{what}: beta must be finite and label_smoothing in [0, 1], got {beta}, {label_smoothing}")
  _check_factor(what, factor)


def compute_preference_loss(logits: torch.Tensor, targets: torch.Tensor, weights: Optional[torch.Tensor],
                            reference_scores: torch.Tensor, beta: float = 0.1, label_smoothing: float = 0.0,
                            loss_normalizing_factor=None):
  """Loss of paired answers by their log ratios against a reference model.

  Rows 2j and 2j + 1 of `logits` [batch, length, vocab] are answers to one prompt, row 2j the preferred one.
  With the score of a row, sum_t weights * log softmax(logits)[targets], and `reference_scores` [batch], the
  scores that the reference model gives (`score_batch` of both models returns such scores),
  margin_j = beta * ((score - reference)_2j - (score - reference)_2j+1), and the loss is the sum (not mean) of
  (1 - label_smoothing) log(1 + exp(-margin)) + label_smoothing log(1 + exp(margin)), over
  `loss_normalizing_factor` if one is given.

  Returns (loss, scores [batch], margins [batch / 2], number of pairs); the loss alone is differentiable, and in
  the logits alone. Tokens of weight 0 do not count, whatever their logits hold, and a pair without any
  other is padding: it counts nowhere. A weighted target outside of the vocabulary gives a NaN loss on the GPU. An
  answer with a target of logit -inf has a score of -inf: rejected, its pair's loss is 0 (without smoothing).

  On the GPU the gradient is computed along with the loss (memory of the logits' size, also where they are a view of
  something larger) for logits in bf16 or fp32, and rounded to their type. A loss that is scaled behind the call has
  its bf16 gradient rounded once more, a `loss_normalizing_factor` comes before the rounding; see
  t5x_b200/ops/token_losses.py."""
  from t5x_b200.ops import token_losses
  what = "compute_preference_loss"
  _check_tokens(what, logits, 3, targets=targets, weights=weights)
  _check_preference(what, logits, reference_scores, beta, label_smoothing, loss_normalizing_factor)
  return token_losses.preference_loss(logits, targets, weights, reference_scores, float(beta),
                                      float(label_smoothing), loss_normalizing_factor)


def preference_loss_from_token_scores(token_scores: torch.Tensor, weights: Optional[torch.Tensor],
                                      reference_scores: torch.Tensor, beta: float = 0.1,
                                      label_smoothing: float = 0.0, loss_normalizing_factor=None):
  """`compute_preference_loss` from log-probabilities of the targets [batch, length], differentiable in them.
  Behind the projection that is fused with its cross entropy, where no logits exist: `token_scores` is minus the
  per-token loss of `functional.logits_cross_entropy` (z-loss and label smoothing 0)."""
  from t5x_b200.ops import token_losses
  what = "preference_loss_from_token_scores"
  _check_tokens(what, token_scores, 2, weights=weights)
  _check_preference(what, token_scores, reference_scores, beta, label_smoothing, loss_normalizing_factor)
  return token_losses.preference_loss(token_scores, None, weights, reference_scores, float(beta),
                                      float(label_smoothing), loss_normalizing_factor)


def _check_policy(what, values, advantages, clip_range, clip_range_high, factor):
  if advantages.shape not in (values.shape[:1], values.shape[:2], (values.shape[0], 1)) or \
      advantages.device != values.device:
    raise ValueError(f"{what}: advantages must be [batch] or [batch, length] = {tuple(values.shape[:2])} on "
                     f"{values.device}, got {tuple(advantages.shape)} on {advantages.device}")
  high = clip_range if clip_range_high is None else clip_range_high
  if not (0.0 <= clip_range <= 1.0 and high >= 0.0):
    raise ValueError(f"{what}: clip_range must lie in [0, 1] and clip_range_high must not be negative, got "
                     f"{clip_range}, {high}")
  _check_factor(what, factor)
  return float(clip_range), float(high)


def compute_policy_loss(logits: torch.Tensor, targets: torch.Tensor, weights: Optional[torch.Tensor],
                        old_token_scores: torch.Tensor, advantages: torch.Tensor,
                        reference_token_scores: Optional[torch.Tensor] = None, clip_range: float = 0.2,
                        clip_range_high: Optional[float] = None, kl_weight: float = 0.0,
                        loss_normalizing_factor=None):
  """Clipped policy loss with a KL term over the tokens of drawn answers.

  With logp = log softmax(logits)[targets] of `logits` [batch, length, vocab], ratio = exp(logp -
  old_token_scores) against the log-probabilities [batch, length] when the answers were drawn, and `advantages`
  ([batch], one for an answer, or [batch, length]), a token's loss is
  -min(advantage * ratio, advantage * clip(ratio, 1 - clip_range, 1 + clip_range_high)) + kl_weight * kl with
  kl = exp(ref - logp) - 1 - (ref - logp) against `reference_token_scores` (None: no such term; with kl_weight 0 it
  is returned and is not part of the loss, whatever its size); clip_range_high is clip_range unless given.
  Log-probabilities are unweighted, as in the `token_scores` that `score_batch` returns for weights of 0 and 1.

  Returns (loss, kl, clipped, weight_sum): the sums (not means) of weights * loss and weights * kl, both over
  `loss_normalizing_factor` if one is given, the weights of the tokens that the clip holds, and all weights. The
  loss alone is differentiable, and in the logits alone. Tokens of weight 0 do not count, whatever is in
  their places. A weighted target outside of the vocabulary gives a NaN loss on the GPU.

  On the GPU loss and gradient take one pass over logits in bf16 or fp32. A loss that is scaled behind the call has its
  bf16 gradient rounded once more, a `loss_normalizing_factor` comes before the rounding; see
  t5x_b200/ops/token_losses.py."""
  from t5x_b200.ops import token_losses
  what = "compute_policy_loss"
  _check_tokens(what, logits, 3, targets=targets, weights=weights, old_token_scores=old_token_scores,
                reference_token_scores=reference_token_scores)
  low, high = _check_policy(what, logits, advantages, clip_range, clip_range_high, loss_normalizing_factor)
  return token_losses.policy_loss(logits, targets, weights, old_token_scores, advantages, reference_token_scores,
                                  low, high, float(kl_weight), loss_normalizing_factor)


def policy_loss_from_token_scores(token_scores: torch.Tensor, weights: Optional[torch.Tensor],
                                  old_token_scores: torch.Tensor, advantages: torch.Tensor,
                                  reference_token_scores: Optional[torch.Tensor] = None, clip_range: float = 0.2,
                                  clip_range_high: Optional[float] = None, kl_weight: float = 0.0,
                                  loss_normalizing_factor=None):
  """`compute_policy_loss` from log-probabilities of the targets [batch, length], differentiable in them (see
  `preference_loss_from_token_scores`)."""
  from t5x_b200.ops import token_losses
  what = "policy_loss_from_token_scores"
  _check_tokens(what, token_scores, 2, weights=weights, old_token_scores=old_token_scores,
                reference_token_scores=reference_token_scores)
  low, high = _check_policy(what, token_scores, advantages, clip_range, clip_range_high, loss_normalizing_factor)
  return token_losses.policy_loss(token_scores, None, weights, old_token_scores, advantages,
                                  reference_token_scores, low, high, float(kl_weight), loss_normalizing_factor)
