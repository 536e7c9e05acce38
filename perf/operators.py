"""What is measured of the operators at the two ends of a fine-tuning step.

* op "preference": the loss of paired answers (log ratios against a reference model) over the logits, with
  its gradient: `losses.compute_preference_loss`;
* op "policy": the clipped policy loss with a KL term over the logits, with its gradient:
  `losses.compute_policy_loss`;
* op "adamw": one AdamW step of all of a model's parameters, moments in 32 bits: `optimizers.adamw`;
* op "adamw8": the same with moments in 8 bits behind a global-norm clip: `optimizers.adamw8`.

With `own` false every operator is computed from elementary tensor operations.
"""
import math

import torch

own = False

CLIP_LOW, CLIP_HIGH, KL_WEIGHT = 0.2, 0.28, 0.05
BETA, SMOOTHING = 0.1, 0.1
LR, B1, B2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
MAX_NORM, STEP, SEED = 1.0, 1000, 7
BLOCK = 256  # values that share a scale in the 8-bit moments

# name: (emb, heads, head_dim, mlp, layers each of encoder and decoder)
SIZES = {
    "tiny": (8, 4, 3, 16, 2),
    "small": (512, 6, 64, 1024, 8),
    "base": (768, 12, 64, 2048, 12),
    "large": (1024, 16, 64, 2816, 24),
}


def _loss(op, rows, length, vocab, dtype):
  return {"op": op, "rows": rows, "length": length, "vocab": vocab, "dtype": dtype}


def _adam(op, size, vocab):
  emb, heads, dim, mlp, layers = SIZES[size]
  return {"op": op, "emb": emb, "heads": heads, "dim": dim, "mlp": mlp, "layers": layers, "vocab": vocab}


def listed():
  cases = [
      # two pairs of short answers of a byte-level model: a call of a few microseconds
      ("preference_bytes", _loss("preference", 4, 48, 384, "float32")),
      # a batch of 32 pairs at the target length of pre-training, logits as a bf16 projection gives them
      ("preference_base", _loss("preference", 64, 114, 32128, "bfloat16")),
      # long answers, fp32 logits as the decoder's own projection gives them; rows of no alignment
      ("preference_long", _loss("preference", 14, 509, 32101, "float32")),
      # byte-level model, long sequences: many short rows
      ("policy_bytes", _loss("policy", 16, 1024, 384, "bfloat16")),
      # a rollout batch of 128 answers
      ("policy_base", _loss("policy", 128, 114, 32128, "bfloat16")),
      # the multilingual vocabulary: one row is a megabyte
      ("policy_multilingual", _loss("policy", 7, 189, 250112, "float32")),
      # the test-sized model: a hundred tensors of a few values each
      ("adamw_tiny", _adam("adamw", "tiny", 384)),
      # T5.1.1 small, all parameters
      ("adamw_small", _adam("adamw", "small", 32128)),
      # T5.1.1 large, all parameters
      ("adamw_large", _adam("adamw", "large", 32128)),
      ("adamw8_tiny", _adam("adamw8", "tiny", 384)),
      ("adamw8_small", _adam("adamw8", "small", 32128)),
      ("adamw8_large", _adam("adamw8", "large", 32128)),
  ]
  return [dict(name=n, **c) for n, c in cases]


def _log_int(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  most = max(work(c)["bytes"] for c in listed())
  while True:
    op = rng.choice(["preference", "policy", "adamw", "adamw8"])
    if op in ("preference", "policy"):
      vocab = rng.choice([384, 32128, 250112, _log_int(rng, 300, 260000), _log_int(rng, 300, 260000)])
      rows = 2 * _log_int(rng, 1, 64) if op == "preference" else _log_int(rng, 1, 128)
      case = _loss(op, rows, _log_int(rng, 1, 1024), vocab, rng.choice(["float32", "bfloat16"]))
      if work(case)["bytes"] <= 1.9e9:
        return case
    else:
      case = {"op": op, "emb": _log_int(rng, 8, 2048), "heads": rng.randint(1, 32), "dim": rng.choice([3, 64, 128]),
              "mlp": _log_int(rng, 16, 5120), "layers": rng.randint(1, 24), "vocab": _log_int(rng, 300, 40000)}
      if work(case)["bytes"] <= most:
        return case


# ----------------------------------------------------------------------------
# Parameters of an encoder-decoder, side by side in flat buffers
# ----------------------------------------------------------------------------
def _shapes(case):
  """Shapes of all parameters in the order of the tree."""
  emb, inner, mlp = case["emb"], case["heads"] * case["dim"], case["mlp"]
  attention = [(emb, inner)] * 3 + [(inner, emb)]
  block = [(emb, mlp)] * 2 + [(mlp, emb)]
  encoder = [(emb,)] + attention + [(emb,)] + block
  decoder = [(emb,)] + attention + [(emb,)] + attention + [(emb,)] + block
  n = case["layers"]
  ends = [(case["heads"], 32), (emb,)]
  return [(case["vocab"], emb)] + encoder * n + ends + decoder * n + ends + [(emb, case["vocab"])]


def _numel(shape):
  return math.prod(shape)


def _blocks(shape):
  return -(-_numel(shape) // BLOCK)


def _views(flat, shapes, starts):
  return {"p%03d" % i: flat[at:at + _numel(s)].view(s) for i, (s, at) in enumerate(zip(shapes, starts))}


def _adam_state(case, seed):
  shapes = _shapes(case)
  counts = torch.tensor([_blocks(s) for s in shapes])
  starts = ((torch.cumsum(counts, 0) - counts) * BLOCK).tolist()  # every tensor begins a block of its own
  total = int(counts.sum()) * BLOCK
  gen = torch.Generator(device="cuda").manual_seed(seed)
  # where a tensor ends inside a block the rest of the block stays zero
  real = torch.zeros(total, dtype=torch.bool, device="cuda")
  for s, at in zip(shapes, starts):
    real[at:at + _numel(s)] = True

  def normal(scale, spread):
    x = torch.randn(total, device="cuda", generator=gen).mul_(scale)
    if spread:  # magnitudes differ from block to block, as they do from layer to layer
      x.view(-1, BLOCK).mul_(torch.exp(spread * torch.randn(total // BLOCK, 1, device="cuda", generator=gen)))
    return x.mul_(real)

  p, g = normal(0.05, 0.0), normal(1e-3, 1.0)
  mu = normal(3e-4, 1.0)
  nu = normal(1e-3, 1.0).square_()
  state = {"case": case, "step": STEP, "p": p, "g": g, "bf16": torch.empty_like(p, dtype=torch.bfloat16)}
  state["bf16"].copy_(p)
  if case["op"] == "adamw":
    state |= {"mu": mu, "nu": nu}
  else:
    state["block_of"] = torch.cat([torch.arange(n) for n in counts.tolist()]).cuda()
    for name, x in (("mu", mu), ("nu", nu)):
      rows = x.view(-1, BLOCK)
      most = rows.abs().amax(1)
      codes = (rows / most.clamp(min=1e-30)[:, None] * 448).to(torch.float8_e4m3fn).view(torch.uint8)
      if name == "nu":
        codes = torch.where((rows > 0) & (codes == 0), torch.ones_like(codes), codes)
      state |= {name: codes.view(-1), name + "_absmax": most}
  if own:
    state["optimizer"] = _optimizer(case, state, shapes, starts)
  return state


def _optimizer(case, state, shapes, starts):
  from t5x_b200 import optax_api, optimizers
  params = _views(state["p"], shapes, starts)
  grads = _views(state["g"], shapes, starts)
  copies = _views(state["bf16"], shapes, starts)
  for name, p in params.items():
    p.bf16 = copies[name]
  tree = lambda d: {"model": d}  # noqa: E731
  if case["op"] == "adamw":
    definition = optimizers.adamw(LR, b1=B1, b2=B2, eps=EPS, weight_decay=DECAY)
  else:
    definition = optimizers.chain([optimizers.clip_by_global_norm(MAX_NORM),
                                   optax_api.adamw8(LR, b1=B1, b2=B2, eps=EPS, weight_decay=DECAY, seed=SEED)])
  optimizer = definition.create(tree(params))
  adam = optimizer.state.param_states
  adam = adam["0"] if case["op"] == "adamw" else adam["1"]["0"]
  adam["count"] = torch.tensor(STEP, dtype=torch.int32)
  for name in ("mu", "nu"):
    adam[name] = tree(_views(state[name], shapes, starts))
    if case["op"] == "adamw8":
      at = [s // BLOCK for s in starts]
      adam[name + "_absmax"] = tree({k: state[name + "_absmax"][a:a + _blocks(s)]
                                     for k, s, a in zip(params, shapes, at)})
  return optimizer, tree(grads)


def _adam_plain(state):
  """m, v, update and weights of AdamW over the flat buffers."""
  case, p, g = state["case"], state["p"], state["g"]
  small = case["op"] == "adamw8"
  mu, nu = state["mu"], state["nu"]
  if small:
    norm = g.double().square().sum().sqrt()
    g = g * torch.clamp(MAX_NORM / (norm + 1e-16), max=1.0).float()
    mu = _values(mu, state["mu_absmax"])
    nu = _values(nu, state["nu_absmax"])
  state["step"] += 1
  t = state["step"]
  m = B1 * mu + (1 - B1) * g
  v = B2 * nu + (1 - B2) * (g * g)
  u = (m / (1 - B1 ** t)) / (torch.sqrt(v / (1 - B2 ** t)) + EPS) + DECAY * p
  p.sub_(LR * u)
  state["bf16"].copy_(p)
  if small:
    noise = _noise(state["block_of"], t)
    _store(state["mu"], state["mu_absmax"], m, noise & 0xFFFF, False)
    _store(state["nu"], state["nu_absmax"], v, noise >> 16, True)
  else:
    state["mu"].copy_(m)
    state["nu"].copy_(v)


def _values(codes, most):
  return (codes.view(torch.float8_e4m3fn).float().view(-1, BLOCK) * (most / 448)[:, None]).view(-1)


def _noise(block_of, step):
  """32 bits for each value, a function of the step and of the value's place in its tensor."""
  low = 0xFFFFFFFF
  key = (SEED * 0x9E3779B1 + step * 0xBB67AE85) & low
  h = block_of[:, None] * BLOCK + torch.arange(BLOCK, device=block_of.device)
  h = ((h + key) * 0x9E3779B1) & low
  h ^= h >> 15
  h = (h * 0x6A09E667) & low
  h ^= h >> 13
  h = (h * 0xBB67AE85) & low
  return h ^ (h >> 16)


def _store(codes, most, x, noise, positive):
  """Rounds x / (largest of the block) * 448 to one of the two e4m3 values next to it, to either with the
  probability that keeps the mean; a second moment that is not zero is not stored as zero."""
  rows = x.view(-1, BLOCK)
  most.copy_(rows.abs().amax(1))
  y = rows.abs() / most.clamp(min=1e-30)[:, None] * 448
  exponent = (torch.frexp(y)[1] - 1).clamp(min=-6)
  gap = torch.ldexp(torch.ones_like(y), exponent - 3)
  y = torch.floor(y / gap + (noise + 0.5) / 65536) * gap
  y = y.clamp(max=448)
  if positive:
    y = torch.where((rows > 0) & (y == 0), 2.0 ** -9, y)
  codes.copy_(torch.copysign(y, rows).to(torch.float8_e4m3fn).view(torch.uint8).view(-1))


def _adam_outputs(state):
  out = {k: state[k] for k in ("p", "bf16", "mu", "nu")}
  if state["case"]["op"] == "adamw8":
    # the stored moments: e4m3 values, and the largest of each block that they are relative to
    out |= {k: state[k].view(torch.float8_e4m3fn) for k in ("mu", "nu")}
    out |= {k: state[k] for k in ("mu_absmax", "nu_absmax")}
  return out


# ----------------------------------------------------------------------------
# Losses
# ----------------------------------------------------------------------------
def _loss_state(case, seed):
  rows, length, vocab = case["rows"], case["length"], case["vocab"]
  gen = torch.Generator(device="cuda").manual_seed(seed)
  dtype = getattr(torch, case["dtype"])
  logits = torch.empty(rows, length, vocab, dtype=dtype, device="cuda")
  targets = torch.randint(0, vocab, (rows, length), device="cuda", generator=gen)
  scores = torch.empty(rows, length, dtype=torch.float64, device="cuda")
  for r in range(rows):
    x = torch.randn(length, vocab, device="cuda", generator=gen).mul_(2)
    # a trained model gives most targets a high probability
    x.scatter_add_(1, targets[r][:, None], 8 + 3 * torch.randn(length, 1, device="cuda", generator=gen))
    logits[r] = x
    x = logits[r].float()
    scores[r] = (x.gather(1, targets[r][:, None])[:, 0] - torch.logsumexp(x, 1)).double()
  # answers of different lengths behind a prompt; weight 1 on the answer
  at = torch.arange(length, device="cuda")
  first = (torch.rand(rows, 1, device="cuda", generator=gen) * 0.15 * length).long()
  last = length - (torch.rand(rows, 1, device="cuda", generator=gen) * 0.25 * length).long()
  weights = ((at >= first) & (at < last)).float()
  state = {"case": case, "logits": logits.requires_grad_(), "targets": targets, "weights": weights}
  if case["op"] == "preference":
    drift = torch.randn(rows, device="cuda", generator=gen) * 5
    state["reference"] = ((scores * weights).sum(1) + drift).float()
  else:
    ratio = torch.exp(torch.randn(rows, length, device="cuda", generator=gen, dtype=torch.float64) * 0.15)
    for border in (1 - CLIP_LOW, 1 + CLIP_HIGH):  # next to a border either side is a right answer: none lies there
      ratio = torch.where((ratio - border).abs() < 1e-3, border + 2e-3, ratio)
    state["old"] = (scores - ratio.log()).float()
    state["reference"] = (scores + torch.randn(rows, length, device="cuda", generator=gen) * 0.3).float()
    state["advantages"] = torch.randn(rows, 1, device="cuda", generator=gen).expand(rows, length).contiguous()
  return state


def _log_probs(logits, targets, visible):
  """Softmax and log-probability of the targets in 32 bits; rows that do not count are taken as zeros."""
  x = torch.where(visible[..., None], logits.detach(), 0).float()
  x = x - x.amax(-1, keepdim=True)
  at = targets[..., None]
  logp = x.gather(-1, at)
  total = x.exp_().sum(-1, keepdim=True)
  return x.div_(total), (logp - total.log())[..., 0]


def _logits_gradient(softmax, targets, by_score, dtype):
  """(d loss / d score) (onehot - softmax)"""
  softmax.mul_(-by_score[..., None])
  return softmax.scatter_add_(-1, targets[..., None], by_score[..., None]).to(dtype)


def _preference_plain(state):
  logits, targets, weights = state["logits"], state["targets"], state["weights"]
  softmax, logp = _log_probs(logits, targets, weights != 0)
  scores = (logp.double() * weights).sum(1)
  against = scores - state["reference"]
  margins = BETA * (against[0::2] - against[1::2])
  real = (weights != 0).any(1).view(-1, 2).any(1)
  # log sigmoid(x) = min(x, 0) - log(1 + exp(-|x|))
  tail = torch.log1p(torch.exp(-margins.abs()))
  loss = (1 - SMOOTHING) * (tail - margins.clamp(max=0)) + SMOOTHING * (tail + margins.clamp(min=0))
  slope = BETA * (1 / (1 + torch.exp(-margins)) - (1 - SMOOTHING)) * real
  by_score = torch.stack([slope, -slope], 1).view(-1, 1) * weights
  grad = _logits_gradient(softmax, targets, by_score.float(), logits.dtype)
  return {"loss": (loss * real).sum().float(), "scores": scores.float(), "margins": (margins * real).float(),
          "pairs": real.sum().float(), "grad": grad}


def _policy_plain(state):
  logits, targets, weights = state["logits"], state["targets"], state["weights"]
  visible = weights != 0
  softmax, logp = _log_probs(logits, targets, visible)
  adv = state["advantages"]
  ratio = torch.exp(logp - state["old"])
  apart = state["reference"] - logp
  gain, held = adv * ratio, adv * ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
  kl = torch.exp(apart) - apart - 1
  clipped = (held < gain).float()
  count = weights.sum()
  by_score = torch.where(visible, weights * (-gain * (1 - clipped) + KL_WEIGHT * (1 - torch.exp(apart))) / count, 0)
  grad = _logits_gradient(softmax, targets, by_score, logits.dtype)
  add = lambda x: (torch.where(visible, x, 0).double() * weights).sum()  # noqa: E731
  return {"loss": (add(KL_WEIGHT * kl - torch.minimum(gain, held)) / count).float(), "kl": (add(kl) / count).float(),
          "clipped": add(clipped).float(), "weight": count, "grad": grad}


def prepare(case, seed):
  return _adam_state(case, seed) if case["op"].startswith("adamw") else _loss_state(case, seed)


def run(state):
  op = state["case"]["op"]
  if op in ("adamw", "adamw8"):
    if own:
      optimizer, grads = state["optimizer"]
      state["optimizer"] = optimizer.apply_gradient(grads), grads
    else:
      _adam_plain(state)
    return _adam_outputs(state)
  if not own:
    return _preference_plain(state) if op == "preference" else _policy_plain(state)
  from t5x_b200 import losses
  logits, weights = state["logits"], state["weights"]
  if op == "preference":
    loss, scores, margins, pairs = losses.compute_preference_loss(
        logits, state["targets"], weights, state["reference"], beta=BETA, label_smoothing=SMOOTHING)
    out = {"loss": loss.detach(), "scores": scores, "margins": margins, "pairs": pairs}
  else:
    loss, kl, clipped, weight = losses.compute_policy_loss(
        logits, state["targets"], weights, state["old"], state["advantages"], state["reference"],
        clip_range=CLIP_LOW, clip_range_high=CLIP_HIGH, kl_weight=KL_WEIGHT,
        loss_normalizing_factor=weights.sum())
    out = {"loss": loss.detach(), "kl": kl, "clipped": clipped, "weight": weight}
  out["grad"] = torch.autograd.grad(loss, logits)[0]
  return out


def work(case):
  op = case["op"]
  if op.startswith("adamw"):
    # read: weights, gradient, both moments; written: weights, their bf16 copy, both moments
    n = sum(_numel(s) for s in _shapes(case))
    return {"bytes": n * (30 if op == "adamw" else 18 + 16 / BLOCK), "flops": n * 16}
  tokens, size = case["rows"] * case["length"], 4 if case["dtype"] == "float32" else 2
  seen = 0.8 * tokens  # tokens of an answer: the logits of the others need not be read, their gradient is zero
  per_token = 12 if op == "preference" else 24
  return {"bytes": (seen + tokens) * case["vocab"] * size + tokens * per_token, "flops": 8 * seen * case["vocab"]}


# ----------------------------------------------------------------------------
# In 64 bits, from the definitions
# ----------------------------------------------------------------------------
def exact(case, seed):
  state = prepare(case, seed)
  if case["op"].startswith("adamw"):
    return _adam_exact(state)
  return _loss_exact(state)


def _adam_exact(state):
  small = state["case"]["op"] == "adamw8"
  n, t = state["p"].numel(), STEP + 1
  factor = 1.0
  if small:
    factor = min(1.0, MAX_NORM / math.sqrt(sum(float(c.double().pow(2).sum()) for c in state["g"].split(1 << 26))))
  out = {"p": torch.empty_like(state["p"])}
  out["bf16"] = None
  for name in ("mu", "nu"):
    out[name] = torch.empty_like(state["p"])
    if small:
      out[name + "_absmax"] = torch.empty_like(state[name + "_absmax"])
  for at in range(0, n, 1 << 26):  # (2 ** 26 is a multiple of the block)
    part = slice(at, min(n, at + (1 << 26)))
    blocks = slice(part.start // BLOCK, part.stop // BLOCK)
    p, g = state["p"][part].double(), state["g"][part].double() * factor
    old = {}
    for name in ("mu", "nu"):
      x = state[name][part]
      if small:
        x = x.view(torch.float8_e4m3fn).double().view(-1, BLOCK) * state[name + "_absmax"][blocks].double()[:, None] / 448
      old[name] = x.double().reshape(-1)
    mu = old["mu"] + (1 - B1) * (g - old["mu"])
    nu = old["nu"] + (1 - B2) * (g ** 2 - old["nu"])
    step = mu / (1 - math.pow(B1, t)) / ((nu / (1 - math.pow(B2, t))) ** 0.5 + EPS)
    out["p"][part] = (p * (1 - LR * DECAY) - LR * step).float()
    for name, x in (("mu", mu), ("nu", nu)):
      if small:
        out[name + "_absmax"][blocks] = x.view(-1, BLOCK).abs().max(1).values.float()
        out[name][part] = _rounded_exact(x, state["block_of"][blocks], t, name).float()
      else:
        out[name][part] = x.float()
  return out


def _rounded_exact(x, block_of, step, name):
  """The e4m3 value that x / (largest of its block) * 448 is rounded to."""
  place = (block_of[:, None] * BLOCK + torch.arange(BLOCK, device=x.device)).reshape(-1)
  h = (place + SEED * 0x9E3779B1 + step * 0xBB67AE85) % 2 ** 32
  for factor, shift in ((0x9E3779B1, 15), (0x6A09E667, 13), (0xBB67AE85, 16)):
    h = h * factor % 2 ** 32
    h = h ^ (h // 2 ** shift)
  h = h % 2 ** 16 if name == "mu" else h // 2 ** 16
  most = x.view(-1, BLOCK).abs().max(1, keepdim=True).values.expand(-1, BLOCK).reshape(-1)
  y = torch.where(most > 0, x.abs() / most * 448, 0)
  below = torch.full_like(y, 2.0 ** -9)  # distance of neighbouring values
  for e in range(-5, 9):
    below = torch.where(y >= 2.0 ** e, 2.0 ** (e - 3), below)
  low = torch.floor(y / below)
  y = (low + (y / below - low + (h + 0.5) / 2 ** 16 >= 1)) * below
  if name == "nu":
    y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
  return y * x.sign()


def _loss_exact(state):
  case, targets, weights = state["case"], state["targets"], state["weights"].double()
  rows, length = case["rows"], case["length"]
  logits = state["logits"].detach()
  seen = [(r, [t for t in range(length) if weights[r, t] != 0]) for r, weights in enumerate([weights.cpu()] * rows)]
  score = torch.zeros(rows, length, dtype=torch.float64, device="cuda")
  for r, at in seen:
    if at:
      score[r, at] = -torch.nn.functional.cross_entropy(logits[r, at].double(), targets[r, at], reduction="none")
  leaf = score.clone().requires_grad_()
  if case["op"] == "preference":
    total = (leaf * weights).sum(1)
    ratio = total - state["reference"].double()
    margin = BETA * (ratio[::2] - ratio[1::2])
    good, bad = torch.nn.functional.softplus(-margin), torch.nn.functional.softplus(margin)
    loss = ((1 - SMOOTHING) * good + SMOOTHING * bad).sum()
    out = {"loss": loss.detach(), "scores": total.detach(), "margins": margin.detach(),
           "pairs": torch.tensor(float(rows // 2))}
  else:
    ratio = (leaf - state["old"].double()).exp()
    adv = state["advantages"].double()
    clip = ratio.clip(1 - CLIP_LOW, 1 + CLIP_HIGH)
    gap = state["reference"].double() - leaf
    kl = gap.exp() - 1 - gap
    mean = lambda x: (x * weights).sum() / weights.sum()  # noqa: E731
    loss = mean(KL_WEIGHT * kl - torch.min(adv * ratio, adv * clip))
    cut = torch.where(adv > 0, ratio > 1 + CLIP_HIGH, (ratio < 1 - CLIP_LOW) & (adv < 0))
    out = {"loss": loss.detach(), "kl": mean(kl).detach(), "clipped": (cut * weights).sum(), "weight": weights.sum()}
  by_score = torch.autograd.grad(loss, leaf)[0]
  grad = torch.zeros_like(logits, dtype=torch.float32)  # rounded once: the steps before it are in 64 bits
  for r, at in seen:
    if at:
      x = torch.nn.functional.softmax(logits[r, at].double(), 1)
      x[torch.arange(len(at)), targets[r, at]] -= 1
      grad[r, at] = (-by_score[r, at][:, None] * x).float()
  out["grad"] = grad
  return out
