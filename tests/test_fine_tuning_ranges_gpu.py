"""The ends of the range of the fine-tuning losses and of AdamW with 8-bit moments on the GPU: large logits and masks of
large values, terms of weight 0 that overflow, answers that cannot be, factors of 0, blocks of the largest and smallest
moments, memory and places of gradients, function transforms."""
import math

import pytest
import torch

from t5x_b200 import losses, optimizers
from tests.test_adamw_group_gpu import adam_of, leaves, to_cpu
from tests.test_token_losses_gpu import call, check, data, oracle_logp

pytestmark = pytest.mark.gpu


LIMIT = 65536.0  # up to here a largest logit's product with log2 e is rounded once for the whole row


def large_rows(vocab, dtype):
  """Rows [18, vocab] and targets: parts of the vocabulary, or all of it, under masks of large negative values; large
  largest values, several of them the same; values on either side of the limit, so that parts of a row lie on both."""
  gen = torch.Generator(device="cuda").manual_seed(vocab)
  rand = lambda n: torch.randn(n, device="cuda", generator=gen)  # noqa: E731
  few = min(300, vocab // 2)
  rows, targets = [], []

  def add(x, t):
    rows.append(x.to(dtype))
    targets.append(t)

  for mask in (-1e7, -1e9, -1e10, -1e20, -1e30):
    x = rand(vocab) * 2
    x[few:] = mask
    add(x, few // 2)  # (in the part that counts)
  for mask in (-1e7, -1e10, -1e30):
    add(torch.full((vocab,), mask, device="cuda"), vocab - 1)
  for big in (1e7, 1e9, 1e10, 1e30):
    x = rand(vocab) * 2
    x[few:few + 5] = big
    add(x, few + 3)
  for middle in (LIMIT, -LIMIT, 1e5, -1e6):
    x = middle + rand(vocab) * 3
    add(x, int(x.argmax()))
  x = rand(vocab) * 2  # parts of several sizes
  for i, v in enumerate((-1e10, -LIMIT, -7e4, -1e6, -1e38)):
    x[vocab * (i + 1) // 7:vocab * (i + 2) // 7] = v
  add(x, 0)
  x = -70000 + rand(vocab) * 3  # lanes of a warp below the limit, the largest above it
  x[vocab // 2] = -65530.0
  add(x, vocab // 2)
  return torch.stack(rows).view(6, 3, vocab), torch.tensor(targets, device="cuda").view(6, 3)


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [64, 4000, 32128, 140001, 250112, 530000])
def test_large_logits(kind, dtype, vocab):
  """Of a warp a row, a block, a cluster, several chunks."""
  d = data(6, 3, vocab, dtype, hidden=0.0)
  d["x"], d["t"] = large_rows(vocab, dtype)
  logp = oracle_logp(d["x"], d["t"])
  assert float(logp.min()) > -40  # (as the tolerances take it)
  d["old"], d["ref"], d["r"] = (logp - 0.1).float(), (logp + 0.1).float(), (logp * d["w"]).sum(1).float() - 1
  x = d["x"].clone().requires_grad_()
  out = call(kind, x, d, None)
  check(kind, out, torch.autograd.grad(out[0], x)[0], d, 1.0)
  with torch.no_grad():
    check(kind, call(kind, d["x"], d, None), None, d, 1.0)


@pytest.mark.parametrize("vocab", [4000, 32128, 250112])
def test_unlikely_targets_among_large_logits(vocab):
  """A target far below the largest logit: its log-probability is their difference, exact in 32 bits here."""
  for big in (1e5, 1e7, 1e10):
    x = torch.zeros(2, 1, vocab, device="cuda")
    x[:, :, vocab // 3] = big
    t = torch.full((2, 1), vocab - 1, device="cuda")
    out = losses.compute_preference_loss(x, t, None, torch.zeros(2, device="cuda"), beta=1e-8)
    assert out[1].tolist() == pytest.approx([-big, -big], rel=2.0 ** -22)


@pytest.mark.parametrize("vocab", [64, 4000, 32128, 250112])
def test_targets_of_the_lowest_logit(vocab):
  """A target at -3e38 among ordinary logits, as likely as it was when it was drawn: ratio 1."""
  x = torch.zeros(2, 1, vocab, device="cuda")
  x[..., 5] = -3e38
  t, old = torch.full((2, 1), 5, device="cuda"), torch.full((2, 1), -3e38, device="cuda")
  x.requires_grad_()
  out = losses.compute_policy_loss(x, t, None, old, torch.ones(2, device="cuda"))
  assert out[0].item() == -2.0
  assert torch.all(torch.autograd.grad(out[0], x)[0][..., 5] == -1.0)


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [101, 4001, 32131, 140005])
def test_large_logits_at_the_ends_of_a_row(kind, dtype, vocab):
  """The values in front of a row's first 16-byte boundary and behind its last, which are added one by one, are its
  largest; the target is one of them, or another."""
  d = data(6, 3, vocab, dtype, hidden=0.0)
  big = torch.zeros(6, 3, vocab + 3, dtype=dtype, device="cuda")
  x = big[..., 3:]
  x.copy_(d["x"])
  middles = torch.tensor([300.3, 1006.7, 30003.7, 60000.3, -30000.6, 65533.9], device="cuda").view(6, 1, 1)
  x.copy_(x.float() + middles)
  for t, at in ((0, 0), (1, vocab - 1), (2, 1)):
    x[:, t, at] = (middles[:, 0, 0] + 9.3).to(dtype)
  d["t"][:, 0], d["t"][:, 1] = 0, vocab - 1
  d["t"][:, 2] = x[:, 2, 2:].argmax(-1) + 2
  d["x"] = x.contiguous()
  logp = oracle_logp(d["x"], d["t"])
  assert float(logp.min()) > -40
  d["old"], d["ref"], d["r"] = (logp - 0.1).float(), (logp + 0.1).float(), (logp * d["w"]).sum(1).float() - 1
  leaf = x.detach().requires_grad_()
  out = call(kind, leaf, d, None)
  check(kind, out, torch.autograd.grad(out[0], leaf)[0], d, 1.0)


@pytest.mark.parametrize("kl_weight", [0.0, 0.1])
@pytest.mark.parametrize("vocab", [0, 2, 3000, 40000])
@pytest.mark.parametrize("host", ["1", "0"])
def test_policy_reference_far_above(kl_weight, vocab, host, monkeypatch):
  """exp(ref - logp) overflows: with weight 0 the term is not part of the loss. (vocab 0: from log-probabilities)"""
  from t5x_b200.ops import native
  monkeypatch.setattr(native, "_host", None if host == "1" else False)
  f = lambda *v: torch.tensor(v, device="cuda").view(2, 1)  # noqa: E731
  rest = (None, f(-100.0, -1.0), torch.ones(2, device="cuda"), f(-1.0, -1.0))
  if vocab:
    x = torch.full((2, 1, vocab), -1000.0, device="cuda")
    x[..., 0], x[..., 1] = 0.0, 100.0
    x[1, 0, 0], x[1, 0, 1] = 100.0, 101.0
    x.requires_grad_()
    out = losses.compute_policy_loss(x, torch.zeros(2, 1, dtype=torch.long, device="cuda"), *rest, kl_weight=kl_weight)
  else:
    x = f(-100.0, -1.0).requires_grad_()
    out = losses.policy_loss_from_token_scores(x, *rest, kl_weight=kl_weight)
  assert out[1].item() == math.inf
  if kl_weight:
    assert out[0].item() == math.inf
    return
  # ratios: 1 (a few roundings of 100 at most), and, with logits, exp(logp + 1) with logp = -log(1 + e)
  second = math.exp(1 - math.log(1 + math.e)) if vocab else 1.0
  assert out[0].item() == pytest.approx(-1.0 - second, abs=6e-5)
  grad = torch.autograd.grad(out[0], x)[0]
  assert torch.all(torch.isfinite(grad))
  if vocab:
    assert grad[0, 0, :2].tolist() == pytest.approx([-1.0, 1.0], abs=6e-5) and torch.all(grad[..., 2:] == 0)
  else:
    assert grad.flatten().tolist() == pytest.approx([-1.0, -1.0], abs=6e-5)


@pytest.mark.parametrize("vocab", [0, 5, 3000, 40000])
def test_policy_of_an_impossible_token(vocab):
  """A token that the model now rules out: ratio 0, and a KL term of infinity where it is asked for."""
  full = lambda v: torch.full((1, 2), v, device="cuda")  # noqa: E731
  rest = (None, full(-1.0), torch.ones(1, device="cuda"), full(-2.0))
  x = torch.zeros(1, 2, max(vocab, 5), device="cuda")
  x[0, 0, 3] = -math.inf
  t = torch.full((1, 2), 3, device="cuda")
  if vocab:
    f = lambda **kw: losses.compute_policy_loss(x, t, *rest, **kw)  # noqa: E731
  else:
    x = x.log_softmax(-1)[..., 3]
    f = lambda **kw: losses.policy_loss_from_token_scores(x, *rest, **kw)  # noqa: E731
  x.requires_grad_()
  out = f()
  other = -min(math.exp(1 - math.log(max(vocab, 5))), 1.2)
  assert out[0].item() == pytest.approx(other, rel=1e-5) and out[1].item() == math.inf
  grad = torch.autograd.grad(out[0], x)[0]
  assert torch.all(grad[0, 0] == 0) and torch.all(torch.isfinite(grad))
  assert f(kl_weight=0.1)[0].item() == math.inf


@pytest.mark.parametrize("vocab", [0, 5, 700, 2000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_preference_of_an_impossible_answer(vocab, dtype):
  """Rejected: margin +inf, loss log(1 + exp(-inf)) = 0, no gradient; preferred: an infinite loss. (vocab 0: from
  log-probabilities)"""
  if vocab == 0 and dtype == torch.bfloat16:
    pytest.skip("log-probabilities are fp32")
  d = data(4, 3, max(vocab, 5), dtype, hidden=0.0)
  r = d["r"]

  def run(row, **kw):
    x = d["x"].detach().clone()
    x[row, 1, d["t"][row, 1]] = -math.inf
    if vocab:
      x.requires_grad_()
      return x, losses.compute_preference_loss(x, d["t"], d["w"], r, **kw)
    x = x.float().log_softmax(-1).gather(-1, d["t"][..., None])[..., 0].requires_grad_()
    return x, losses.preference_loss_from_token_scores(x, d["w"], r, **kw)

  x, (loss, scores, margins, pairs) = run(1)
  clean = losses.compute_preference_loss(d["x"][2:].contiguous(), d["t"][2:], d["w"][2:], r[2:])[0]
  assert loss.item() == pytest.approx(clean.item(), rel=1e-5) and pairs.item() == 2
  assert scores[1].item() == -math.inf and margins[0].item() == math.inf and math.isfinite(margins[1].item())
  grad = torch.autograd.grad(loss, x)[0]
  assert torch.all(grad[:2] == 0) and torch.all(torch.isfinite(grad)) and torch.any(grad[2:] != 0)
  assert run(1, label_smoothing=0.1)[1][0].item() == math.inf
  x, out = run(0)
  assert out[0].item() == math.inf and out[2][0].item() == -math.inf
  assert torch.all(torch.isfinite(torch.autograd.grad(out[0], x)[0]))
  assert math.isfinite(run(0, label_smoothing=1.0)[1][0].item())


@pytest.mark.parametrize("host", ["1", "0"])
def test_normalizing_factor_of_zero(host, monkeypatch):
  """What tensor operations give, whether the factor lies on the host or on the device."""
  from t5x_b200.ops import native
  monkeypatch.setattr(native, "_host", None if host == "1" else False)
  d = data(2, 3, 50, torch.float32, hidden=0.0)
  for factor in (0.0, 0, torch.tensor(0.0), torch.tensor(0.0, device="cuda")):
    assert call("preference", d["x"], d, factor)[0].item() == math.inf
    assert math.isnan(call("policy", d["x"], dict(d, w=0 * d["w"]), factor)[0].item())


def chain8(**kw):
  return optimizers.chain([optimizers._adamw8(1e-2, weight_decay=0.0, **kw)])


def same_step(gpu, g, **kw):
  """A step on the GPU and, from the same state, by the tensor operations on the CPU: the same weights, scales, and
  codes but for draws beside their border (a few in 2^16, see test_8_bits_match_the_tensor_operations)."""
  cpu = chain8(**kw).create(to_cpu(gpu.target))
  cpu.state.param_states = to_cpu(gpu.state.param_states)
  gpu, cpu = gpu.apply_gradient(g), cpu.apply_gradient(to_cpu(g))
  for p, q in zip(leaves(gpu.target), leaves(cpu.target)):
    assert torch.allclose(p.cpu(), q, rtol=2 ** -22, atol=1e-2 * 2 ** -18)
  a, b = adam_of(gpu), adam_of(cpu)
  for name in ("mu", "nu"):
    for x, y in zip(leaves(a[name + "_absmax"]), leaves(b[name + "_absmax"])):
      assert torch.allclose(x.cpu(), y, rtol=2 ** -20, atol=0, equal_nan=True)
    for x, y in zip(leaves(a[name]), leaves(b[name])):
      d = (x.cpu().int() - y.int()).abs()
      assert int(d.max()) <= 1 and int((d > 0).sum()) <= 4
  return gpu


@pytest.mark.parametrize("host", ["1", "0"])
@pytest.mark.parametrize("largest", [1.8e19, 1.2e19, 1e10, 1.0, 1e-10, 1e-15, 3e-18, 1e-18, 4e-19])
def test_moments_at_the_ends_of_the_range(largest, host, monkeypatch):
  """nu = g^2 / 2 up to 1.6e38 and down to 8e-38; every value of it is a normal number of 32 bits. Steps with no gradient
  follow: what was stored is read back, and never as zero where it was above zero."""
  from t5x_b200.ops import native
  monkeypatch.setattr(native, "_host", None if host == "1" else False)
  gen = torch.Generator(device="cuda").manual_seed(1)
  g = torch.rand(5000, device="cuda", generator=gen) * 0.5 + 0.5
  g = g * torch.where(torch.rand(5000, device="cuda", generator=gen) < 0.5, -1.0, 1.0) * largest
  kw = dict(b2=0.5, eps=1e-30, seed=4)
  gpu = chain8(**kw).create({"a": {"w": torch.zeros(5000, device="cuda"), "v": torch.zeros(5000, device="cuda")}})
  gpu = same_step(gpu, {"a": {"w": g, "v": g.flip(0).contiguous()}}, **kw)
  nu = leaves(adam_of(gpu)["nu"])[0]
  # (a quarter of the largest or more, and 56, an eighth, is 0x66; the scale is 2^-100 at least)
  assert int(nu.min()) >= (0x66 if largest > 1.3e-15 else 1)
  none = torch.zeros(5000, device="cuda")
  for _ in range(3):
    before = [p.clone() for p in leaves(gpu.target)]
    gpu = same_step(gpu, {"a": {"w": none, "v": none}}, **kw)
    assert all(float((p - b).abs().max()) < 0.02 for p, b in zip(leaves(gpu.target), before))


def test_small_moments_beside_a_small_largest():
  """A block whose smallest code stands for less than a normal number of 32 bits: nothing in it reads as zero."""
  g = torch.full((2000,), 4.5e-18, device="cuda")  # nu 2e-38
  g[::256] = 1e-15  # nu 1e-33, a code of 1 is 4e-39
  kw = dict(eps=1e-30, seed=4)
  gpu = chain8(**kw).create({"w": torch.zeros(2000, device="cuda")})
  gpu = same_step(gpu, {"w": g}, **kw)
  for _ in range(3):
    before = gpu.target["w"].clone()
    gpu = same_step(gpu, {"w": torch.zeros(2000, device="cuda")}, **kw)
    assert int(adam_of(gpu)["nu"]["w"].min()) > 0
    assert float((gpu.target["w"] - before).abs().max()) < 0.05


@pytest.mark.parametrize("size", [600, 601])
def test_overflowing_second_moment_shows(size):
  """A square beyond 32 bits: its block is NaN when it is read back, as behind a NaN, not a step of 0 for good."""
  w = {"w": torch.ones(size, device="cuda")}
  opt = optimizers.adamw8(1e-2, weight_decay=0.0).create(w)
  g = torch.ones(size, device="cuda")
  g[300] = 1e20
  opt = opt.apply_gradient({"w": g})
  assert torch.all(torch.isfinite(opt.target["w"]))
  assert torch.isnan(adam_of(opt)["nu_absmax"]["w"]).tolist() == [False, True, False]
  opt = opt.apply_gradient({"w": torch.ones(size, device="cuda")})
  assert torch.isnan(opt.target["w"]).nonzero().flatten().tolist() == list(range(256, 512))


@pytest.mark.parametrize("host", ["1", "0"])
@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [501, 4001, 40003])
def test_gradient_of_a_view_takes_the_memory_of_its_values(kind, dtype, vocab, host, monkeypatch):
  """The last tokens of much longer rows, a part of a much larger vocabulary: values as those of a copy, memory of the
  values' own size (and up to 16 bytes a row)."""
  from t5x_b200.ops import native
  monkeypatch.setattr(native, "_host", None if host == "1" else False)
  d = data(4, 5, vocab, dtype)
  big = torch.empty(4, 60, 2 * vocab + 3, dtype=dtype, device="cuda")
  big[:, 50:55, 7:7 + vocab] = d["x"]
  for view in (big[:, 50:55, 7:7 + vocab].detach(), big[:, 50:55, 7:7 + vocab].detach()[::2], d["x"].detach()):
    e = d if view.shape[0] == 4 else {k: v[::2].contiguous() for k, v in d.items()}
    e = dict(e, x=view.contiguous())
    leaf = view.requires_grad_()
    call(kind, leaf, e, None)  # (what is allocated once)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call(kind, leaf, e, None)
    grad = torch.autograd.grad(out[0], leaf, retain_graph=True)[0]
    peak = torch.cuda.max_memory_allocated() - before
    # twice (the graph is kept), 16 bytes a row, each rounded up by the allocator; scratch
    rows = view.shape[0] * 5
    assert peak <= 2 * (view.numel() * view.element_size() + 16 * rows + 16) + (4 << 20) and grad.shape == view.shape
    check(kind, out, grad, e, 1.0)
    assert torch.equal(torch.autograd.grad(out[0], leaf)[0], grad)


def test_gradient_beyond_32_bits():
  """More than 2^31 values; the tokens that count lie at the end."""
  length, vocab, few = 34000, 32128, 3
  d = data(2, few, vocab, torch.bfloat16, hidden=0.0)
  x = torch.empty(2, length, vocab, dtype=torch.bfloat16, device="cuda")
  assert x[1].storage_offset() + (length - few) * vocab > 2 ** 31
  x[:, -few:] = d["x"]
  pad = lambda v, fill=0.0: torch.nn.functional.pad(v, (length - few, 0), value=fill)  # noqa: E731
  for kind in ("preference", "policy"):
    e = dict(d, **{k: pad(d[k]) for k in ("w", "old", "adv", "ref")}, t=pad(d["t"], 0))
    leaf = x.detach().requires_grad_()
    out = call(kind, leaf, e, None)
    grad = torch.autograd.grad(out[0], leaf)[0]
    check(kind, out, grad[:, -few:], d, 1.0)
    assert not torch.any(grad[0, :-few]) and not torch.any(grad[1, :-few])
    del leaf, out, grad


@pytest.mark.parametrize("host", ["1", "0"])
def test_function_transforms(host, monkeypatch):
  """Under `torch.func` the statements run, which can be transformed."""
  from t5x_b200.ops import native
  monkeypatch.setattr(native, "_host", None if host == "1" else False)
  d = data(4, 3, 50, torch.float32)
  for kind in ("preference", "policy"):
    loss = lambda v: call(kind, v, d, 2.0)[0]  # noqa: E731
    leaf = d["x"].clone().requires_grad_()
    want = torch.autograd.grad(loss(leaf), leaf)[0]
    got = torch.func.grad(loss)(d["x"])
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-6)
    along = torch.randn_like(d["x"])
    slope = torch.func.jvp(loss, (d["x"],), (along,))[1]
    assert float(slope) == pytest.approx(float((want * along).sum()), rel=1e-4, abs=1e-5)


@pytest.mark.parametrize("host", ["1", "0"])
@pytest.mark.parametrize("seed", [2 ** 64 - 3, 2 ** 63, -7, 2 ** 32 + 1])
def test_seeds_of_any_size(seed, host, monkeypatch):
  """The rounding depends on the seed modulo 2^32; seeds of 64 bits without a sign are common."""
  from t5x_b200.ops import native
  monkeypatch.setattr(native, "_host", None if host == "1" else False)
  g = torch.randn(3000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
  states = []
  for s in (seed, seed % 2 ** 32, seed % 2 ** 32 + 1):
    opt = optimizers.adamw8(1e-2, seed=s).create({"w": torch.ones(3000, device="cuda")})
    states.append(adam_of(opt.apply_gradient({"w": g}))["mu"]["w"])
  assert torch.equal(states[0], states[1]) and not torch.equal(states[0], states[2])
  cpu = optimizers.adamw8(1e-2, seed=seed).create({"w": torch.ones(3000)}).apply_gradient({"w": g.cpu()})
  assert int((adam_of(cpu)["mu"]["w"] != states[0].cpu()).sum()) <= 4
