"""Plain PyTorch statements of every op: the numerical oracle and the CPU path.

Each function restates the math of the corresponding reference op in fp32 (citations
give the file in the reference project whose behaviour is matched). The CUDA kernels in
``csrc/`` are tested against these.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F

NEG_MASK = -1e10  # additive mask value (t5x/examples/t5/layers.py:306-318)


def rmsnorm(x: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
  """T5 "LayerNorm": no mean subtraction, no bias, fp32 statistics (layers.py:683-702)."""
  xf = x.float()
  ms = (xf * xf).mean(dim=-1, keepdim=True)
  return (xf * torch.rsqrt(ms + eps) * scale.float()).to(x.dtype)


def gelu_tanh(x: torch.Tensor) -> torch.Tensor:
  return F.gelu(x, approximate="tanh")


ACTIVATIONS = {
    "relu": F.relu,
    "gelu": gelu_tanh,  # flax.linen.gelu defaults to the tanh approximation
    "linear": lambda x: x,
    "silu": F.silu,
    "swish": F.silu,
    "tanh": torch.tanh,
    "sigmoid": torch.sigmoid,
}


def relative_position_bucket(relative_position: torch.Tensor, bidirectional: bool = True,
                             num_buckets: int = 32, max_distance: int = 128) -> torch.Tensor:
  """T5 relative-position bucket of `k_pos - q_pos` (layers.py:581-625)."""
  ret = torch.zeros_like(relative_position)
  n = -relative_position
  if bidirectional:
    num_buckets //= 2
    ret = ret + (n < 0).to(n.dtype) * num_buckets
    n = n.abs()
  else:
    n = n.clamp(min=0)
  max_exact = num_buckets // 2
  is_small = n < max_exact
  eps = torch.finfo(torch.float32).eps
  val_if_large = max_exact + (
      torch.log(n.to(torch.float32) / max_exact + eps) / math.log(max_distance / max_exact) *
      (num_buckets - max_exact)).to(n.dtype)
  val_if_large = val_if_large.clamp(max=num_buckets - 1)
  return ret + torch.where(is_small, n, val_if_large)


def relative_position_bias(table: torch.Tensor, qlen: int, klen: int, bidirectional: bool,
                           num_buckets: int = 32, max_distance: int = 128,
                           q_offset: int = 0) -> torch.Tensor:
  """[heads, qlen, klen] bias from a [heads, num_buckets] table (layers.py:627-677)."""
  dev = table.device
  ctx = torch.arange(q_offset, q_offset + qlen, device=dev)[:, None]
  mem = torch.arange(klen, device=dev)[None, :]
  buckets = relative_position_bucket(mem - ctx, bidirectional, num_buckets, max_distance)
  return table[:, buckets]  # [H, q, k]


class PrefixLMMask:
  """Visibility of a prefix LM in factored form: key k is visible to query q when
  (k <= q, or both lie inside the prefix) and both are real tokens of the same packed segment
  (the semantics of make_decoder_mask with decoder_causal_attention,
  t5x/examples/t5/layers.py:842-924). `bool()` gives the dense [B, 1, L, L] mask, so the object
  can stand wherever a dense `extra_mask` is accepted; the flash kernels use the per-token
  vectors and never build the dense form."""

  def __init__(self, in_prefix: torch.Tensor, valid: torch.Tensor,
               segment_ids: Optional[torch.Tensor] = None):
    self.in_prefix, self.valid, self.segment_ids = in_prefix.bool(), valid.bool(), segment_ids

  def bool(self) -> torch.Tensor:
    b, l = self.valid.shape
    pos = torch.arange(l, device=self.valid.device)
    vis = (pos[None, :] <= pos[:, None])[None].expand(b, l, l)
    vis = vis | (self.in_prefix[:, :, None] & self.in_prefix[:, None, :])
    vis = vis & self.valid[:, :, None] & self.valid[:, None, :]
    if self.segment_ids is not None:
      vis = vis & (self.segment_ids[:, :, None] == self.segment_ids[:, None, :])
    return vis[:, None]

  def token_codes(self):
    """(query codes, key codes) int32 [B, L] for the kernels: the segment id (1 when unpacked)
    in the low 30 bits, bit 30 set inside the prefix; padding queries carry a segment id that no
    key has, so their rows see nothing."""
    seg = self.segment_ids.to(torch.int32) if self.segment_ids is not None else \
        torch.ones_like(self.valid, dtype=torch.int32)
    pre = self.in_prefix.to(torch.int32) << 30
    k_codes = seg | pre
    q_codes = torch.where(self.valid, seg, torch.full_like(seg, 0x3FFFFFFE)) | pre
    return q_codes.contiguous(), k_codes.contiguous()


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
              bias: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
              causal: bool = False, q_segment_ids: Optional[torch.Tensor] = None,
              kv_segment_ids: Optional[torch.Tensor] = None,
              extra_mask: Optional[torch.Tensor] = None,
              float32_logits: bool = True) -> torch.Tensor:
  """softmax(q k^T + bias + mask) v with no 1/sqrt(d) (T5 folds it into the init).

  q [B, Lq, H, D]; k, v [B, Lk, H, D]; bias [H or 1, Lq, Lk] (relative positions);
  key_mask [B, Lk] bool (True = attend). Masked logits get -1e10, so a fully masked
  row yields a uniform distribution, never NaN (layers.py:52-129).
  `extra_mask` [B, 1 or H, Lq, Lk] bool is and-ed in (prefix-LM blocks).
  """
  dt = torch.float32 if float32_logits else q.dtype
  logits = torch.einsum("bqhd,bkhd->bhqk", q.to(dt), k.to(dt))
  if bias is not None:
    logits = logits + bias.to(dt)[None]
  B, H, Lq, Lk = logits.shape
  mask = None

  def _and(m, new):
    return new if m is None else (m & new)

  if key_mask is not None:
    mask = _and(mask, key_mask[:, None, None, :].bool())
  if causal:
    qi = torch.arange(Lq, device=q.device)[:, None] + (Lk - Lq)
    ki = torch.arange(Lk, device=q.device)[None, :]
    mask = _and(mask, (ki <= qi)[None, None])
  if q_segment_ids is not None and kv_segment_ids is not None:
    mask = _and(mask, (q_segment_ids[:, None, :, None] == kv_segment_ids[:, None, None, :]))
  if extra_mask is not None:
    mask = _and(mask, extra_mask.bool())
  if mask is not None:
    # Additive, as in the reference (mask -> bias of 0 / -1e10 that is summed with the logits):
    # a masked logit equals -1e10 in fp32 and the softmax gradient still reaches q and k.
    logits = logits + torch.where(mask, 0.0, NEG_MASK).to(logits.dtype)
  probs = torch.softmax(logits.float(), dim=-1).to(v.dtype)
  return torch.einsum("bhqk,bkhd->bqhd", probs, v)


def cross_entropy_with_logits(logits: torch.Tensor, targets: torch.Tensor, z_loss: float):
  """Per-position (loss incl. z-loss, z-loss term) for soft `targets` (t5x/losses.py:62-95)."""
  logits = logits.float()
  lse = torch.logsumexp(logits, dim=-1)
  log_softmax = logits - lse[..., None]
  loss = -(targets * log_softmax).sum(-1)
  total_z = z_loss * lse * lse
  return loss + total_z, total_z


def label_smoothing_constants(vocab: int, label_smoothing: float):
  confidence = 1.0 - label_smoothing
  low_confidence = (1.0 - confidence) / (vocab - 1)
  normalizing_constant = -(confidence * math.log(confidence) +
                           (vocab - 1) * low_confidence * math.log(low_confidence + 1e-20))
  return confidence, low_confidence, normalizing_constant


def token_cross_entropy(logits: torch.Tensor, targets: torch.Tensor, z_loss: float = 0.0,
                        label_smoothing: float = 0.0):
  """Per-token (ce+z - normalizing const, z term, lse, argmax) for integer targets
  (t5x/losses.py:132-193 without the weighting/normalisation step)."""
  vocab = logits.shape[-1]
  confidence, low_confidence, norm_const = label_smoothing_constants(vocab, label_smoothing)
  lf = logits.float()
  lse = torch.logsumexp(lf, dim=-1)
  tl = lf.gather(-1, targets[..., None]).squeeze(-1)
  if label_smoothing > 0:
    soft_dot = confidence * tl + low_confidence * (lf.sum(-1) - tl)
  else:
    soft_dot = tl
  z = z_loss * lse * lse
  loss = lse - soft_dot + z - norm_const
  return loss, z, lse, lf.argmax(-1)


_DROPOUT_GENERATORS: dict = {}


def set_dropout_seed(seed: Optional[int]) -> None:
  """Seeds the generators used by `dropout` (one per device); None returns to global RNG.
  Also restarts the numbering of dropout sites used by the in-kernel masks."""
  _DROPOUT_GENERATORS.clear()
  _DROPOUT_SITE[0] = 0
  if seed is not None:
    _DROPOUT_GENERATORS["seed"] = int(seed)


_DROPOUT_SITE = [0]


def dropout_seed() -> Optional[int]:
  """The seed set by `set_dropout_seed`, or None."""
  return _DROPOUT_GENERATORS.get("seed")


def next_dropout_site() -> int:
  """A number that is different for every dropout call since the last `set_dropout_seed`:
  together with the seed it names the mask of that call (the in-kernel generator is keyed by
  (seed, site, element))."""
  _DROPOUT_SITE[0] += 1
  return _DROPOUT_SITE[0]


def dropout_site_state() -> int:
  return _DROPOUT_SITE[0]


def set_dropout_site_state(n: int) -> None:
  """Restores the site counter (recomputation of a checkpointed block must draw the masks of
  its first pass)."""
  _DROPOUT_SITE[0] = int(n)


def _dropout_generator(device) -> Optional[torch.Generator]:
  if "seed" not in _DROPOUT_GENERATORS:
    return None
  key = str(device)
  if key not in _DROPOUT_GENERATORS:
    g = torch.Generator(device=device)
    g.manual_seed(_DROPOUT_GENERATORS["seed"])
    _DROPOUT_GENERATORS[key] = g
  return _DROPOUT_GENERATORS[key]


def dropout(x: torch.Tensor, rate: float, training: bool, broadcast_dims=(),
            generator: Optional[torch.Generator] = None) -> torch.Tensor:
  """Dropout whose mask is shared along `broadcast_dims` (flax nn.Dropout semantics)."""
  if not training or rate == 0.0:
    return x
  if generator is None and dropout_seed() is not None:
    # one generator per call, keyed by (step seed, call number): a block that is recomputed in
    # the backward pass (rematerialisation) restores the call counter and so draws the masks
    # of its first pass again, as the in-kernel generator on the GPU does
    generator = torch.Generator(device=x.device)
    generator.manual_seed((dropout_seed() * 1000003 + next_dropout_site()) % (2 ** 63 - 1))
  shape = list(x.shape)
  for d in broadcast_dims:
    shape[d] = 1
  keep = 1.0 - rate
  mask = torch.rand(shape, device=x.device, generator=generator) < keep
  return torch.where(mask, x / keep, torch.zeros_like(x))


# ----------------------------------------------------------------------------
# Losses of preference and policy fine-tuning
# ----------------------------------------------------------------------------
def _wide(t: torch.Tensor) -> torch.Tensor:
  return t if t.dtype == torch.float64 else t.float()


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor,
                    weights: Optional[torch.Tensor] = None) -> torch.Tensor:
  """log softmax(logits)[target] in 32 bits; 0 for tokens of weight 0, whatever their logits hold."""
  if weights is None:
    return _wide(logits).log_softmax(-1).gather(-1, targets[..., None].long())[..., 0]
  seen = weights != 0
  x = torch.where(seen[..., None], _wide(logits), torch.zeros((), dtype=_wide(logits).dtype, device=logits.device))
  at = torch.where(seen, targets.long(), torch.zeros_like(targets, dtype=torch.long))
  logp = x.log_softmax(-1).gather(-1, at[..., None])[..., 0]
  return torch.where(seen, logp, torch.zeros_like(logp))


def _over_normalizer(loss: torch.Tensor, normalizer) -> torch.Tensor:
  if normalizer is None:
    return loss
  return loss / (normalizer.detach().to(loss.device) if isinstance(normalizer, torch.Tensor) else normalizer)


def policy_loss(logp, weights, old, advantages, reference, clip_low, clip_high, kl_weight, normalizer):
  """(loss, kl, clipped, weight) from log-probabilities [B, L]:
  sum w (kl_weight kl - min(A rho, A clip(rho, 1 - clip_low, 1 + clip_high))) / normalizer with
  rho = exp(logp - old) and kl = exp(reference - logp) - 1 - (reference - logp)."""
  logp = _wide(logp)
  w = torch.ones_like(logp) if weights is None else weights.detach().to(logp.dtype)
  seen, zero = w != 0, torch.zeros((), dtype=logp.dtype, device=logp.device)
  adv = advantages.detach().to(logp.dtype)
  adv = (adv[:, None] if adv.dim() == 1 else adv).expand(logp.shape)
  pick = lambda t: torch.where(seen, t.detach().to(logp.dtype), zero)  # noqa: E731
  logp, adv = torch.where(seen, logp, zero), pick(adv)
  ratio = torch.exp(logp - pick(old))
  gain, held = adv * ratio, adv * ratio.clamp(1.0 - clip_low, 1.0 + clip_high)
  each, kl = -torch.minimum(gain, held), torch.zeros_like(logp)
  if reference is not None:
    apart = pick(reference) - logp
    kl = torch.where(torch.isposinf(apart), apart, torch.expm1(apart) - apart)
    if kl_weight != 0:  # (of a term that only is reported an overflow stays out of the loss)
      each = each + kl_weight * kl
  total = lambda t: torch.where(seen, t * w, zero).sum(dtype=torch.float64)  # noqa: E731
  back = logp.dtype
  return (_over_normalizer(total(each), normalizer).to(back), _over_normalizer(total(kl.detach()), normalizer).to(back),
          total((held < gain).to(back)).to(back), w.sum(dtype=torch.float64).to(back))


def preference_loss(logp, weights, reference, beta, label_smoothing, normalizer):
  """(loss, scores, margins, pairs) from log-probabilities [B, L], rows 2j (preferred) and 2j + 1 a pair:
  scores = sum_t w logp, margin = beta ((s_2j - r_2j) - (s_2j+1 - r_2j+1)),
  loss = sum (1 - e) log(1 + exp(-margin)) + e log(1 + exp(margin)), over the normalizer. Pairs without a
  token of weight are padding."""
  logp = _wide(logp)
  w = torch.ones_like(logp) if weights is None else weights.detach().to(logp.dtype)
  seen, zero = w != 0, torch.zeros((), dtype=torch.float64, device=logp.device)
  scores = torch.where(seen, logp.double() * w, zero).sum(-1)
  real = seen.any(-1).view(-1, 2).any(-1)
  apart = scores - torch.where(real.repeat_interleave(2), reference.detach().double(), zero)
  margins = torch.where(real, beta * (apart[0::2] - apart[1::2]), zero)
  # (a side of weight 0 may be infinite: the answer that is not preferred cannot be)
  sides = [w * F.softplus(m) for w, m in ((1.0 - label_smoothing, -margins), (label_smoothing, margins)) if w != 0]
  loss = sum(sides[1:], sides[0])
  back = logp.dtype
  return (_over_normalizer(torch.where(real, loss, zero).sum(), normalizer).to(back), scores.detach().to(back),
          margins.detach().to(back), real.sum().to(back))


# ----------------------------------------------------------------------------
# Numbers in 8 bits
# ----------------------------------------------------------------------------
def codes_of(real: torch.Tensor, whole, most: torch.Tensor) -> torch.Tensor:
  """The code of real * whole / most: the exact quotient rounded to the nearest whole number (ties to even; in 64 bits it
  cannot round to the other side of a border), 0 where it is none."""
  q = torch.round(real.double() * whole / most.double())
  return torch.nan_to_num(q, nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127, 127).to(torch.int8)


def quantize_rows(x: torch.Tensor):
  """(codes int8, fp32 largest |x|) of each row of x [rows, k]; a code c stands for c * largest / 127."""
  x = x.float()
  most = x.abs().amax(1) if x.shape[0] else x.new_zeros(0)
  return codes_of(x, 127, most[:, None]), most


def linear8(x, codes, absmax, residual=None):
  """x [rows, k] times weights in 8 bits [n, k]: x in 8 bits too, scaled by row; sums of whole numbers, rounded once."""
  cx, most = quantize_rows(x)
  y = cx.double() @ codes.double().t()  # (exact)
  y = y * (most.double() / 127)[:, None] * (absmax.double() / 127)
  return (y if residual is None else y + residual.double()).to(x.dtype)


def _cache8_block(cache) -> int:
  return cache["cached_key"].shape[2] // cache["key_absmax"].shape[2]


def _cache8_index(cache) -> torch.Tensor:
  """Tokens held, by row."""
  b, _, slots, _ = cache["cached_key"].shape
  return cache["cache_index"].long().clamp(0, slots).expand(b)


def cache8_append(cache, key, value, lengths=None) -> None:
  """Tokens key, value [B, L, H, D] behind those that the rows hold (lengths [B]: so many of the L). A block of tokens
  that gets some has the largest absolute value of what it holds and gets, and its codes are rounded again."""
  b, h, slots, dim = cache["cached_key"].shape
  block, count, at = _cache8_block(cache), key.shape[1], _cache8_index(cache)
  slot = torch.arange(slots, device=at.device)
  place = slot - at[:, None]  # of the new token, for each slot [B, slots]
  fresh = count if lengths is None else lengths.long().clamp(0, count)[:, None]
  new, old = (place >= 0) & (place < fresh), place < 0
  by_block = lambda t: t.view(b, -1, block).any(2)[:, None]  # noqa: E731
  spread = lambda t: t.repeat_interleave(block, 2)[..., None]  # noqa: E731
  touched, keeps = by_block(new), by_block(old)
  for name, x in (("key", key), ("value", value)):
    codes, most = cache["cached_" + name], cache[name + "_absmax"]
    x = x.float().transpose(1, 2).gather(2, place.clamp(0, count - 1)[:, None, :, None].expand(b, h, slots, dim))
    x = torch.where(new[:, None, :, None], x, torch.zeros_like(x))
    before = torch.where(keeps, most, torch.zeros_like(most))
    after = torch.maximum(before, x.abs().reshape(b, h, -1, block * dim).amax(3))
    again = torch.where(spread(before == after), codes, codes_of(spread(before), codes, spread(after)))
    again = torch.where((old[:, None] & touched.repeat_interleave(block, 2))[..., None], again, codes)
    codes.copy_(torch.where(new[:, None, :, None], codes_of(x, 127, spread(after)), again))
    most.copy_(torch.where(touched, after, most))
  if "token_weight" in cache:
    cache["token_weight"].masked_fill_(new[:, None], 0.0)
  if "token_position" in cache:
    where = (slot + cache["dropped"].long()[:, None]).to(torch.int32)
    cache["token_position"].copy_(torch.where(new[:, None], where[:, None], cache["token_position"]))


def cache8_values(cache, name: str, dtype=torch.float32) -> torch.Tensor:
  """What the codes of "key" or "value" stand for, [B, H, slots, D]."""
  scale = (cache[name + "_absmax"].to(dtype) / 127).repeat_interleave(_cache8_block(cache), 2)
  return cache["cached_" + name].to(dtype) * scale[..., None]


def cache8_attention(query, cache, appended=0, bias_table=None, num_buckets=32, max_distance=128, key_mask=None,
                     causal=True, scale=1.0):
  """softmax(scale q k + bias) v over a cache in 8 bits; query [B, L, heads * group, D]. Of the tokens that a row holds the
  last `appended` are this call's; with `causal` the queries are the last L of all. A query that sees nothing has zeros."""
  wide = torch.promote_types(query.dtype, torch.float32)
  b, h, slots, dim = cache["cached_key"].shape
  count, group = query.shape[1], query.shape[2] // h
  index = _cache8_index(cache)
  end = (index + appended).clamp(max=slots)[:, None, None]
  slot = torch.arange(slots, device=query.device)
  own = (index + appended - count)[:, None] + torch.arange(count, device=query.device)  # slots of the queries [B, L]
  seen = (slot < end).expand(b, count, slots)
  if causal:
    seen = seen & (slot <= own[..., None])
  if key_mask is not None:
    shown = F.pad(key_mask.bool(), (0, slots - key_mask.shape[1]))
    seen = seen & shown[:, None]
  seen = seen[:, None, None]  # [B, 1, 1, L, slots]
  q = query.to(wide).view(b, count, h, group, dim)
  s = torch.einsum("blhgd,bhsd->bhgls", q, cache8_values(cache, "key", wide)) * scale
  if bias_table is not None:
    place, at = slot.expand(b, h, slots), own
    if "token_position" in cache:
      place, at = cache["token_position"].long(), own + cache["dropped"].long()[:, None]
    buckets = relative_position_bucket(place[:, :, None] - at[:, None, :, None], False, num_buckets, max_distance)
    table = bias_table.to(wide)[:h * group].view(h, 1, group, -1)
    s = s + table.expand(h, count, group, -1)[None].expand(b, -1, -1, -1, -1).transpose(2, 3).gather(
        4, buckets[:, :, None].expand(b, h, group, count, slots))
  s = s.masked_fill(~seen, -math.inf)
  top = s.amax(4, keepdim=True)
  p = torch.exp(s - torch.where(torch.isneginf(top), torch.zeros_like(top), top))
  p = torch.where(seen, p, torch.zeros_like(p))
  total = p.sum(4, keepdim=True)
  p = torch.where(total == 0, torch.zeros_like(p), p / total)
  if "token_weight" in cache:
    cache["token_weight"] += p.sum((2, 3)).to(torch.float32)
  v = cache8_values(cache, "value", wide)[:, :, None, None]
  # (what is hidden counts for nothing, whatever its block holds)
  visible = seen.expand_as(p)
  out = torch.einsum("bhgls,bhsd->blhgd", p, torch.nan_to_num(v[:, :, 0, 0], nan=0.0, posinf=0.0, neginf=0.0))
  broken = ~torch.isfinite(v[:, :, 0, 0, :, :1])  # whole blocks
  poisoned = (visible & broken[:, :, None, None, :, 0]).any(4)  # [B, H, group, L]
  out = torch.where(poisoned.permute(0, 3, 1, 2)[..., None], torch.full_like(out, math.nan), out)
  return out.reshape(query.shape).to(query.dtype)


def cache8_evict(cache, into, keep: int, recent: int):
  """Kept slots [B, H, keep] (-1 behind them): the last `recent` tokens and those of the largest weight (NaN above all, ties
  to the lowest slot), in order; `into` gets them, its tokens behind them stay as they were."""
  b, h, slots, dim = cache["cached_key"].shape
  held = _cache8_index(cache)[:, None, None]
  slot = torch.arange(slots, device=held.device)
  rank = torch.argsort(torch.argsort(torch.where(slot < held - recent, cache["token_weight"].double(), -math.inf), dim=2,
                                     descending=True, stable=True), dim=2)
  # where a weight is -inf itself, places before the last ones still come first by the stable order
  stays = (slot < held) & ((held <= keep) | (slot >= held - recent) | (rank < keep - recent))
  kept = torch.where(stays, slot, slots).sort(2).values
  kept = F.pad(kept, (0, max(0, keep - slots)), value=slots)[..., :keep]
  there, source = kept < slots, kept.clamp(max=slots - 1)
  block, old_block = _cache8_block(into), _cache8_block(cache)
  blocks = -(-keep // block)
  grown = lambda t, v: F.pad(t, (0, blocks * block - keep), value=v).view(b, h, blocks, block)  # noqa: E731
  for name in ("key", "value"):
    most = cache[name + "_absmax"].gather(2, source // old_block)
    after = grown(torch.where(there, most, torch.zeros_like(most)), 0.0).amax(3)
    each = after.repeat_interleave(block, 2)[..., :keep, None]
    codes = cache["cached_" + name].gather(2, source[..., None].expand(-1, -1, -1, dim))
    codes = torch.where(most[..., None] == each, codes, codes_of(most[..., None], codes, each))
    to = into["cached_" + name][:, :, :keep]
    to.copy_(torch.where(there[..., None], codes, to))
    to = into[name + "_absmax"][:, :, :blocks]
    to.copy_(torch.where(grown(there, False).any(3), after, to))
  positions = cache.get("token_position", slot.to(torch.int32).expand(b, h, slots))
  for name, t in (("token_weight", cache["token_weight"]), ("token_position", positions)):
    to = into[name][:, :, :keep]
    to.copy_(torch.where(there, t.gather(2, source), to))
  index = cache["cache_index"].clamp(min=0).expand(b)
  left = index.clamp(max=min(keep, slots))
  before = cache["dropped"] if "token_position" in cache else torch.zeros_like(index)
  into["cache_index"].copy_(left)
  into["dropped"].copy_(before + index - left)
  return torch.where(there, kept, -1).to(torch.int32)
