"""Losses of preference and policy fine-tuning with their gradients.

On CUDA, over bf16 or fp32 logits or fp32 log-probabilities, the kernels of csrc/token_losses.cu
compute the loss and, where a gradient will be wanted, the gradient in the same pass; backward
multiplies it by the gradient of the loss (which leaves it alone where that is 1). Anything else
runs the PyTorch statements in :mod:`t5x_b200.ops.reference`, as do calls under a function transform.

The arguments are those of `t5x_b200.losses`, which checks them.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from t5x_b200.ops import functional as F
from t5x_b200.ops import native
from t5x_b200.ops import reference as ref


def _native_ok(values: torch.Tensor, targets: Optional[torch.Tensor]) -> bool:
  """Whether the kernels take the values. (A function transform, a forward-mode level or a trace sees into the statements,
  not into the kernels.)"""
  types = (torch.float32,) if targets is None else (torch.bfloat16, torch.float32)
  return values.is_cuda and values.dtype in types and values.numel() > 0 and not F._transformed()


def _rows_apart(logits: torch.Tensor) -> torch.Tensor:
  """The logits as the kernels take them: values of a row side by side, rows in order and apart."""
  (b, l, v), (sb, st, sv) = logits.shape, logits.stride()
  if (sv == 1 or v == 1) and (l == 1 or st >= v) and (b == 1 or sb >= (l - 1) * st + v):
    return logits
  return logits.contiguous()


def _like(values: torch.Tensor) -> torch.Tensor:
  """Memory for the gradient of `values`: of their size, whatever their strides, at the same place of 16 bytes, so that
  the kernel's wide accesses fall on the same values of both."""
  strides = native.loss_gradient_strides(values) if values.dim() == 3 else values.stride()
  behind = values.data_ptr() % 16 // values.element_size()
  span = sum((n - 1) * s for n, s in zip(values.shape, strides)) + 1
  flat = torch.empty(span + behind, dtype=values.dtype, device=values.device)
  return flat.as_strided(values.shape, strides, behind)


def _times(grad: torch.Tensor, factor: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
  """The saved gradient times the gradient of the loss; None where there is none."""
  if factor is None:
    return None
  return native.scale_gradient(grad, factor.detach().float().reshape(1), keep=F._graph_is_kept())


def _loss(ctx, name, values, targets, *args):
  """The outputs of the kernels' loss `name`; its gradient is kept with the graph where it will be wanted."""
  want = not isinstance(ctx, F._NoGraph) and ctx.needs_input_grad[0]
  values = values.contiguous() if targets is None else _rows_apart(values)
  grad = _like(values) if want else None
  out = getattr(native, name)(values, grad, targets, *args)
  ctx.save_for_backward(grad)
  ctx.mark_non_differentiable(*out[1:])
  ctx.set_materialize_grads(False)
  return out


def _run(fn, name, *args):
  """The loss by the compiled host path, which makes its own node of the graph, or else by `fn`."""
  host = native.host()
  if host is not None:
    out = getattr(host, name)(*args)
    if out:
      return tuple(out)
  return F._apply(fn, *args)


class _PolicyFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, values, *args):
    return _loss(ctx, "policy_loss", values, *args)

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, by, *_):
    return (_times(ctx.saved_tensors[0], by),) + (None,) * 10


class _PreferenceFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, values, *args):
    return _loss(ctx, "preference_loss", values, *args)

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, by, *_):
    return (_times(ctx.saved_tensors[0], by),) + (None,) * 7


def _plain(t: Optional[torch.Tensor], dtype=torch.float32) -> Optional[torch.Tensor]:
  """A contiguous tensor of the type, without its graph."""
  if t is None:
    return None
  if t.requires_grad:
    t = t.detach()
  return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _divisor(factor, device):
  """(1 / factor, None), or (1, the factor as a device scalar)."""
  if factor is None:
    return 1.0, None
  if isinstance(factor, torch.Tensor) and factor.numel() == 1 and factor.device.type != "cpu":
    return 1.0, _plain(factor.reshape(1).to(device))
  factor = float(factor)
  return 1.0 / factor if factor else math.copysign(math.inf, factor), None


def policy_loss(values, targets, weights, old, advantages, reference, clip_low, clip_high, kl_weight,
                normalizer):
  """(loss, kl, clipped, weight); values: logits [B, L, V], or log-probabilities [B, L] with targets
  None."""
  if not _native_ok(values, targets):
    logp = values if targets is None else ref.token_log_probs(values, targets, weights)
    return ref.policy_loss(logp, weights, old, advantages, reference, clip_low, clip_high, kl_weight,
                           normalizer)
  scale, divisor = _divisor(normalizer, values.device)
  return _run(_PolicyFn, "policy_loss", values, _plain(targets, torch.int64), _plain(weights), _plain(old),
              _plain(advantages), _plain(reference), clip_low, clip_high, kl_weight, scale, divisor)


def preference_loss(values, targets, weights, reference, beta, label_smoothing, normalizer):
  """(loss, scores, margins, pairs); values as in `policy_loss`, rows 2j and 2j + 1 a pair."""
  if not _native_ok(values, targets):
    logp = values if targets is None else ref.token_log_probs(values, targets, weights)
    return ref.preference_loss(logp, weights, reference, beta, label_smoothing, normalizer)
  scale, divisor = _divisor(normalizer, values.device)
  return _run(_PreferenceFn, "preference_loss", values, _plain(targets, torch.int64), _plain(weights),
              _plain(reference), beta, label_smoothing, scale, divisor)
