"""A step of preference and of policy fine-tuning as a user writes it: reference scores from `score_batch`, the loss
over the model's logits or behind the fused projection, its backward pass, clipping and AdamW with 8-bit moments."""
import pytest
import torch

from t5x_b200 import losses, optax_api, optimizers

pytestmark = pytest.mark.gpu


def build():
  from t5x_b200 import models, trainer
  from t5x_b200.data import vocabularies
  from t5x_b200.models import base
  from t5x_b200.models.t5 import network
  torch.manual_seed(0)
  module = network.Transformer(network.T5Config(
      vocab_size=2112, dtype="bfloat16", emb_dim=128, num_heads=2, num_encoder_layers=1, num_decoder_layers=1,
      head_dim=64, mlp_dim=256, mlp_activations=("gelu", "linear"), dropout_rate=0.0), device="cuda")
  vocab = vocabularies.PassThroughVocabulary(2112)
  definition = optimizers.chain([optimizers.clip_by_global_norm(0.5),
                                 optax_api.adamw8(1e-3, weight_decay=0.01, seed=3)])
  model = models.EncoderDecoderModel(module, vocab, vocab, definition)
  params = base.module_param_tree(module)
  trainer.attach_compute_buffers(params, bf16_copy=True, main_grad=True)
  return model, params


def make_batch(model, params):
  gen = torch.Generator().manual_seed(1)
  enc = torch.randint(3, 2000, (6, 40), generator=gen)
  tgt = torch.randint(3, 2000, (6, 24), generator=gen)
  tgt[1, 15:] = 0
  tgt[4:] = 0  # a pair of padding
  b = {"encoder_input_tokens": enc, "decoder_target_tokens": tgt,
       "decoder_input_tokens": torch.cat([torch.zeros(6, 1, dtype=torch.long), tgt[:, :-1]], 1),
       "decoder_loss_weights": (tgt > 0).float()}
  b = {k: v.cuda() for k, v in b.items()}
  scores, more = model.score_batch(params, b, return_intermediates=True)
  b["reference"] = scores + torch.tensor([1.0, -2.0, 0.5, 3.0, 0.0, 0.0], device="cuda")
  b["old"] = more["decoder"]["token_scores"][0]
  b["advantages"] = torch.tensor([1.0, -0.5, 2.0, 0.25, 1.0, 1.0], device="cuda")
  return b


def logits_of(model, params, b):
  from t5x_b200.ops import functional as F
  hidden, weight, scale = model._compute_hidden(params, b)
  assert scale == 1.0
  return F.linear(hidden, weight)


def loss_of(model, params, b, kind, route):
  from t5x_b200.ops import functional as F
  targets, w = b["decoder_target_tokens"], b["decoder_loss_weights"]
  factor = w.sum()
  if route == "logits":
    values = (logits_of(model, params, b), targets)
    calls = losses.compute_preference_loss, losses.compute_policy_loss
  else:
    hidden, weight, scale = model._compute_hidden(params, b)
    values = (-F.logits_cross_entropy(hidden, weight, targets, logits_scale=scale)[0],)
    calls = losses.preference_loss_from_token_scores, losses.policy_loss_from_token_scores
  if kind == "preference":
    return calls[0](*values, w, b["reference"], beta=0.2, loss_normalizing_factor=factor)
  return calls[1](*values, w, b["old"], b["advantages"], b["old"] - 0.1, kl_weight=0.1, loss_normalizing_factor=factor)


def slopes(logp, b, kind):
  """dloss / dlogp of each token in 64 bits."""
  w = b["decoder_loss_weights"].double()
  if kind == "preference":
    d = (logp * w).sum(1) - b["reference"].double()
    k = -0.2 * torch.sigmoid(-0.2 * (d[0::2] - d[1::2]))
    return torch.stack([k, -k], 1).view(-1, 1) * w / w.sum()
  rho = torch.exp(logp - b["old"].double())
  a = b["advantages"].double()[:, None]
  held = a * rho.clamp(0.8, 1.2) < a * rho
  return (torch.where(held, 0.0, -a * rho) + 0.1 * (1 - torch.exp(b["old"].double() - 0.1 - logp))) * w / w.sum()


def gradients(params):
  from t5x_b200 import trainer
  from t5x_b200.utils import tree
  flat = tree.flatten_dict(params)
  out = {k: g.clone() for k, g in trainer._collect_grads(flat).items()}
  trainer._begin_step(flat)
  return out


@pytest.mark.parametrize("route", ["logits", "scores"])
@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_gradients_of_the_weights(kind, route):
  """Against the model's own backward pass from the formula's gradient of the logits: what differs is the rounding of
  that gradient to the logits' type and, behind the fused projection, logits that are not rounded at all, 2^-9 and some
  2^-7 of an element, and the order of sums: 3 % of a tensor's norm as for the model's bf16 gradients elsewhere."""
  from t5x_b200 import trainer
  from t5x_b200.ops import native
  from t5x_b200.utils import tree
  model, params = build()
  b = make_batch(model, params)
  trainer._begin_step(tree.flatten_dict(params))
  before = native.launch_count()
  out = loss_of(model, params, b, kind, route)
  out[0].backward()
  assert native.launch_count() > before
  native.check_status()
  got = gradients(params)
  logits = logits_of(model, params, b)
  x = logits.detach().double()
  logp = torch.log_softmax(x, -1)
  onehot = torch.nn.functional.one_hot(b["decoder_target_tokens"], x.shape[-1])
  slope = slopes(logp.gather(-1, b["decoder_target_tokens"][..., None])[..., 0], b, kind)
  logits.backward((slope[..., None] * (onehot - logp.exp())).to(logits.dtype))
  want = gradients(params)
  assert any(float(v.norm()) > 0 for v in want.values())
  for k, v in want.items():
    assert float((got[k].double() - v.double()).norm()) <= 3e-2 * float(v.double().norm()) + 1e-9, k


def test_steps_with_8_bit_moments():
  """Two steps, preference and then policy: from the gradients that the losses left, each agrees with the statements of
  the same optimizer on the CPU (see the tests of that optimizer for the tolerances; the norm is a sum of some 500,000
  squares)."""
  from t5x_b200 import trainer
  from t5x_b200.utils import tree
  model, params = build()
  b = make_batch(model, params)
  optimizer = model.optimizer_def.create(params)
  for kind in ("preference", "policy"):
    trainer._begin_step(tree.flatten_dict(params))
    out = loss_of(model, params, b, kind, "logits")
    out[0].backward()
    grads = tree.unflatten_dict(gradients(params))
    cpu = model.optimizer_def.create(to_cpu(optimizer.target))
    cpu.state.param_states = to_cpu(optimizer.state.param_states)
    old = {k: v.detach().clone() for k, v in tree.flatten_dict(optimizer.target).items()}
    optimizer, cpu = optimizer.apply_gradient(grads), cpu.apply_gradient(to_cpu(grads))
    for k, q in tree.flatten_dict(cpu.target).items():
      p = tree.flatten_dict(optimizer.target)[k]
      assert torch.isfinite(p).all() and (not float(tree.flatten_dict(grads)[k].norm()) or not torch.equal(p, old[k]))
      assert torch.allclose(p.detach().cpu(), q.detach(), rtol=2 ** -20, atol=1e-3 * 2 ** -14), k
      if getattr(p, "bf16", None) is not None:
        assert torch.equal(p.bf16, p.detach().to(torch.bfloat16))


def to_cpu(t):
  if isinstance(t, dict):
    return {k: to_cpu(v) for k, v in t.items()}
  return t.detach().cpu().clone() if isinstance(t, torch.Tensor) else t
