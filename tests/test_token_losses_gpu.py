"""The kernels of the preference and policy losses against the formulas in 64 bits, over sizes, types, strides, masks
and odd values, and the ways in which autograd reaches them."""
import math

import pytest
import torch

from t5x_b200 import losses

pytestmark = pytest.mark.gpu

BETA, SMOOTH, LOW, HIGH, KL = 0.1, 0.1, 0.2, 0.3, 0.05


def data(batch, length, vocab, dtype, seed=0, hidden=0.3):
  gen = torch.Generator(device="cuda").manual_seed(seed)
  rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
  x = (rand(batch, length, vocab) * 2).to(dtype)
  t = torch.randint(0, vocab, (batch, length), device="cuda", generator=gen)
  w = (torch.rand(batch, length, device="cuda", generator=gen) >= hidden).float()
  w = w * (0.5 + torch.rand(batch, length, device="cuda", generator=gen))
  logp = oracle_logp(x, t)
  old = (logp - rand(batch, length) * 0.3).float()
  # the ratio lies beside the clip's borders, where either answer is right, nowhere
  ratio = torch.exp(logp - old.double())
  for border in (1 - LOW, 1 + HIGH):
    near = (ratio - border).abs() < 1e-3
    old = torch.where(near, (logp - math.log(border + 2e-3)).float(), old)
  return dict(x=x, t=t, w=w, r=((logp * w).sum(1) + rand(batch) * 3).float(), old=old, adv=rand(batch, length),
              ref=(logp + rand(batch, length) * 0.3).float())


def oracle_logp(x, t):
  x = x.detach().double()
  x = x - x.amax(-1, keepdim=True)
  return (x.gather(-1, t[..., None]) - x.exp().sum(-1, keepdim=True).log())[..., 0]


def oracle(kind, d, factor):
  """Values and the slope of each token in 64 bits; the gradient follows from the slope."""
  x, t, w = d["x"], d["t"], d["w"].double()
  logp = torch.where(w != 0, oracle_logp(x, t), 0.0)
  if kind == "preference":
    s = (logp * w).sum(1)
    real = (w != 0).any(1).view(-1, 2).any(1)
    m = torch.where(real, BETA * ((s - d["r"])[0::2] - (s - d["r"])[1::2]), 0.0)
    loss = torch.where(real, -(1 - SMOOTH) * torch.nn.functional.logsigmoid(m) -
                       SMOOTH * torch.nn.functional.logsigmoid(-m), 0.0).sum() / factor
    k = torch.where(real, BETA * (torch.sigmoid(m) - 1 + SMOOTH), 0.0) / factor
    return [loss, s, m, real.sum().double()], torch.stack([k, -k], 1).view(-1, 1) * w
  rho = torch.exp(logp - d["old"].double())
  a = d["adv"].double()
  gain, held = a * rho, a * rho.clamp(1 - LOW, 1 + HIGH)
  apart = d["ref"].double() - logp
  kl = torch.exp(apart) - 1 - apart
  slope = torch.where(held < gain, 0.0, -gain) + KL * (1 - torch.exp(apart))
  add = lambda v: torch.where(w != 0, v * w, 0.0).sum()  # noqa: E731
  return [add(KL * kl - torch.minimum(gain, held)) / factor, add(kl) / factor, add((held < gain).double()),
          w.sum()], torch.where(w != 0, slope * w, 0.0) / factor


def call(kind, x, d, factor):
  if kind == "preference":
    return losses.compute_preference_loss(x, d["t"], d["w"], d["r"], beta=BETA, label_smoothing=SMOOTH,
                                          loss_normalizing_factor=factor)
  return losses.compute_policy_loss(x, d["t"], d["w"], d["old"], d["adv"], d["ref"], clip_range=LOW,
                                    clip_range_high=HIGH, kl_weight=KL, loss_normalizing_factor=factor)


def check(kind, out, grad, d, factor):
  x, t = d["x"], d["t"]
  batch, length, vocab = x.shape
  want, slope = oracle(kind, d, float(factor))
  # A log-probability: a thread's sum of up to vocab / 32 terms (one rounding each), the exponentials 2^-21, the
  # difference to the largest and its product 2^-24 * 20 each.
  off = (vocab / 32 + 16) * 2.0 ** -24 + 2.0 ** -21 + 40 * 2.0 ** -24
  tokens = float((d["w"].double() * off).sum())  # of all sums over tokens
  size = [1.0] * 4
  if kind == "preference":
    per = float(d["w"].sum(1).max()) * off + 1e-6 * float(want[1].abs().max())
    allow = [BETA * 2 * per * batch / float(factor), per, BETA * 2 * per + 1e-6, 0.0]
    # the slope moves by beta / 4 of what the margin does, and with it dlogits
    d_slope = BETA / float(factor) * d["w"].double() * (BETA / 4 * 2 * per + 2.0 ** -20)
  else:
    big = float((d["adv"].abs().max() * 4 + 4))
    allow = [big * tokens / float(factor), big * tokens / float(factor), 0.0, 1e-6 * float(want[3])]
    d_slope = d["w"].double() / float(factor) * big * (off + 2.0 ** -20)
  for got, w, a, s in zip(out, want, allow, size):
    assert got.dtype == torch.float32
    assert torch.all((got.double() - w).abs() <= a + 2.0 ** -22 * w.abs()), (got, w, a)
  if grad is None:
    return
  assert grad.shape == x.shape and grad.dtype == x.dtype
  half = torch.finfo(x.dtype).eps / 2
  for b in range(batch):  # (row by row: 64-bit logits of a large vocabulary are large)
    p = torch.softmax(x[b].detach().double(), -1)
    g = -slope[b][:, None] * p
    g.scatter_add_(1, t[b][:, None], slope[b][:, None])
    hot = p.scatter(1, t[b][:, None], 1.0)
    a = half * g.abs() * 1.01 + hot * (d_slope[b] + slope[b].abs() * 2 * off)[:, None] + 1e-37
    g = torch.where((d["w"][b] != 0)[:, None], g, 0.0)
    assert torch.all((grad[b].double() - g).abs() <= a), float(((grad[b].double() - g).abs() - a).max())


SHAPES = [(2, 1, 1), (2, 1, 2), (2, 3, 7), (4, 5, 31), (2, 2, 33), (6, 9, 384), (4, 3, 385), (2, 4, 2047), (2, 3, 2048),
          (4, 3, 2049), (2, 5, 4099), (2, 7, 32128), (4, 2, 32101), (2, 2, 65537), (2, 1, 250112), (2, 3, 530000),
          (10, 2, 8193), (6, 50, 16390), (2, 2, 131071), (2, 600, 40),
          (40, 33, 100), (2, 40, 12345), (8, 150, 4100), (4, 300, 9001), (6, 120, 32101), (10, 100, 20000),
          (4, 25, 250112)]


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(kind, dtype, shape):
  d = data(*shape, dtype, seed=shape[2])
  factor = 1.0 if shape[0] == 2 else 5.0
  x = d["x"].requires_grad_()
  out = call(kind, x, d, factor if factor != 1.0 else None)
  grad = torch.autograd.grad(out[0], x)[0]
  check(kind, out, grad, d, factor)
  with torch.no_grad():
    again = call(kind, x, d, torch.tensor(factor, device="cuda"))
  for u, v in zip(again[1:], out[1:]):
    assert torch.equal(u, v) or kind == "policy"
  check(kind, again, None, d, factor)


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("vocab", [384, 5003, 32128])
def test_the_same_call_twice_gives_the_same_bits(kind, vocab):
  d = data(8, 37, vocab, torch.bfloat16)
  x = d["x"].requires_grad_()
  runs = []
  for _ in range(3):
    out = call(kind, x, d, None)
    runs.append([*[o.detach() for o in out], torch.autograd.grad(out[0], x)[0]])
  for r in runs[1:]:
    assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cut", ["length", "batch", "vocab", "odd start", "transposed", "expanded"])
def test_strides(kind, dtype, cut):
  """Views of larger logits: rows at any place of 16 bytes, rows and batches apart, and what is copied first."""
  d = data(4, 6, 2100, dtype)
  x = d["x"]
  if cut == "length":
    big = torch.randn(4, 9, 2100, device="cuda").to(dtype)
    big[:, 1:7] = x
    view = big[:, 1:7]
  elif cut == "batch":
    big = torch.randn(8, 6, 2100, device="cuda").to(dtype)
    big[::2] = x
    view = big[::2]
  elif cut == "vocab":
    big = torch.randn(4, 6, 2111, device="cuda").to(dtype)
    big[..., 3:2103] = x
    view = big[..., 3:2103]
  elif cut == "odd start":
    flat = torch.zeros(x.numel() + 5, device="cuda", dtype=dtype)
    flat[5:] = x.reshape(-1)
    view = flat[5:].view(x.shape)
  elif cut == "transposed":
    view = x.transpose(0, 1).contiguous().transpose(0, 1)
  else:
    x = x[:, :, :1].expand(4, 6, 2100)
    view, d = x, dict(d, x=x.contiguous())
  view = view.detach().requires_grad_()
  d = dict(d, x=view.detach().contiguous())
  if cut == "expanded":
    logp = oracle_logp(d["x"], d["t"])
    d["old"], d["ref"] = logp.float() - 0.05, logp.float() + 0.1
  out = call(kind, view, d, None)
  check(kind, out, torch.autograd.grad(out[0], view)[0], d, 1.0)


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("vocab", [100, 2500])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_places_hold_anything(kind, vocab, bad):
  d = data(6, 5, vocab, torch.float32)
  d["w"][0:2] = 0  # a pair of padding
  d["w"][2] = 0    # an answer without tokens
  seen = d["w"] != 0
  clean = call(kind, d["x"].clone().requires_grad_(), d, None)
  x = torch.where(seen[..., None], d["x"], bad).requires_grad_()
  e = dict(d, t=torch.where(seen, d["t"], 1 << 40), r=d["r"].clone())
  e["r"][:2] = bad
  for name in ("old", "adv", "ref"):
    e[name] = torch.where(seen, d[name], bad)
  out = call(kind, x, e, None)
  grad = torch.autograd.grad(out[0], x)[0]
  for a, b in zip(out, clean):
    assert torch.equal(a, b)
  assert torch.all(grad[~seen] == 0) and torch.all(torch.isfinite(grad)) and torch.any(grad[seen] != 0)
  check(kind, out, None, d, 1.0)


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_nothing_visible(kind):
  d = data(4, 3, 50, torch.float32, hidden=2.0)
  assert float(d["w"].sum()) == 0
  x = d["x"].requires_grad_()
  out = call(kind, x, d, None)
  assert float(out[0]) == 0 and float(out[3]) == 0
  assert torch.all(torch.autograd.grad(out[0], x)[0] == 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [64, 4000])
def test_masked_vocabulary_and_extreme_logits(dtype, vocab):
  """-inf and the type's lowest value on parts of the vocabulary, rows at the edges of the range, rows of one value."""
  low = torch.finfo(dtype).min
  d = data(6, 4, vocab, dtype)
  x = d["x"]
  hide = torch.rand(x.shape, device="cuda") < 0.5
  hide.scatter_(2, d["t"][..., None], False)
  x[0] = x[0].masked_fill(hide[0], -math.inf)
  x[1] = x[1].masked_fill(hide[1], low)
  x[2] = low
  x[3] = torch.finfo(dtype).max
  x[4, :2] = 0
  x[5] = x[5] * 0.25 + 1000
  d["x"] = x
  logp = oracle_logp(x, d["t"])
  d["old"], d["ref"], d["r"] = (logp - 0.1).float(), (logp + 0.1).float(), (logp * d["w"]).sum(1).float() - 1
  for kind in ("preference", "policy"):
    leaf = x.clone().requires_grad_()
    out = call(kind, leaf, d, None)
    check(kind, out, torch.autograd.grad(out[0], leaf)[0], d, 1.0)


@pytest.mark.parametrize("vocab", [64, 4000])
@pytest.mark.parametrize("what", ["nan", "inf", "all -inf", "target high", "target negative"])
def test_bad_visible_values_make_the_loss_nan(vocab, what):
  for kind in ("preference", "policy"):
    d = data(4, 4, vocab, torch.float32, hidden=0.0)
    if what == "nan":
      d["x"][1, 2, vocab // 2] = math.nan
    elif what == "inf":
      d["x"][1, 2, vocab // 2] = math.inf
    elif what == "all -inf":
      d["x"][1, 2] = -math.inf
    else:
      d["t"][1, 2] = vocab if what == "target high" else -1
    x = d["x"].requires_grad_()
    out = call(kind, x, d, None)
    assert math.isnan(float(out[0]))
    grad = torch.autograd.grad(out[0], x)[0]
    assert torch.all(torch.isfinite(grad[2:]))  # the other pair's, the other answers'


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_scaled_and_graph_kept(kind, dtype):
  d = data(4, 5, 3001, dtype)
  x = d["x"].requires_grad_()
  plain = torch.autograd.grad(call(kind, x, d, None)[0], x)[0]
  loss = call(kind, x, d, None)[0]
  first = torch.autograd.grad(loss * 3.0, x, retain_graph=True)[0]
  assert torch.equal(first, (plain.float() * 3.0).to(dtype))  # (one rounding more)
  second = torch.autograd.grad(loss, x, retain_graph=True)[0]
  third = torch.autograd.grad(loss * 0.5, x)[0]
  assert torch.equal(second, plain) and torch.equal(third, (plain.float() * 0.5).to(dtype))
  assert torch.equal(first, (plain.float() * 3.0).to(dtype))


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("shape", [(2, 1), (4, 7), (64, 114), (2, 5000), (600, 3)])
def test_from_token_scores(kind, shape):
  gen = torch.Generator(device="cuda").manual_seed(1)
  rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
  logp = -rand(*shape).abs()
  w = (torch.rand(*shape, device="cuda", generator=gen) > 0.2).float()
  ratio = torch.exp(rand(*shape) * 0.2)
  ratio = torch.where((ratio - 1 + LOW).abs() < 1e-3, 0.9, torch.where((ratio - 1 - HIGH).abs() < 1e-3, 1.0, ratio))
  old, adv, ref, r = logp - ratio.log(), rand(shape[0]), logp + 0.1 * rand(*shape), rand(shape[0])
  logp = torch.where(w != 0, logp, math.nan)

  def both(v, ww, rr, oo, aa, ff):
    if kind == "preference":
      return losses.preference_loss_from_token_scores(v, ww, rr, label_smoothing=0.2, loss_normalizing_factor=7.0)
    return losses.policy_loss_from_token_scores(v, ww, oo, aa, ff, LOW, HIGH, KL, loss_normalizing_factor=7.0)

  a = logp.clone().requires_grad_()
  b = logp.double().cpu().requires_grad_()
  got = both(a, w, r, old, adv, ref)
  want = both(b, *[t.double().cpu() for t in (w, r, old, adv, ref)])
  for u, v in zip(got, want):
    torch.testing.assert_close(u.double().cpu(), v, rtol=2e-6, atol=2e-6)
  ga, gb = torch.autograd.grad(got[0], a)[0], torch.autograd.grad(want[0], b)[0]
  torch.testing.assert_close(ga.double().cpu(), gb, rtol=4e-6, atol=1e-8)


def test_other_types_take_the_statements():
  d = data(4, 3, 20, torch.float32)
  for dtype in (torch.float16, torch.float64):
    x = d["x"].to(dtype).requires_grad_()
    out = call("preference", x, dict(d, x=x), None)
    assert torch.autograd.grad(out[0], x)[0].dtype == dtype


def test_another_stream_and_capture():
  for kind in ("preference", "policy"):
    d = data(6, 9, 3000, torch.bfloat16)
    x = d["x"].requires_grad_()
    out = call(kind, x, d, None)
    want = [*[o.detach().clone() for o in out], torch.autograd.grad(out[0], x)[0]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
      out = call(kind, x, d, None)
      got = [*[o.detach() for o in out], torch.autograd.grad(out[0], x)[0]]
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    del out
    x = x.detach().requires_grad_()  # (no eager graph of the leaf lives while its backward pass is captured)
    for _ in range(2):  # two graphs; each has memory of its own
      graph = torch.cuda.CUDAGraph()
      with torch.cuda.graph(graph):
        out = call(kind, x, d, None)
        kept = [*[o.detach() for o in out], torch.autograd.grad(out[0], x)[0]]
        del out
      graphs.append((graph, kept))
    for _ in range(3):
      for graph, _ in graphs:
        graph.replay()
    for _, kept in graphs:
      assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_offsets_beyond_32_bits():
  """Rows that begin behind 2^31 values."""
  length, vocab = 3, 1 << 20
  big = torch.empty(2 * 1100, vocab, dtype=torch.bfloat16, device="cuda")
  d = data(2, length, vocab, torch.bfloat16)
  view = big.as_strided((2, length, vocab), (2100 * vocab, 40 * vocab, 1))
  view.copy_(d["x"])
  for kind in ("preference", "policy"):
    leaf = view.detach().requires_grad_()
    out = call(kind, leaf, d, None)
    check(kind, out, torch.autograd.grad(out[0], leaf)[0], d, 1.0)


@pytest.mark.parametrize("host", ["1", "0"])
@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_loss_in_a_larger_graph(kind, host, monkeypatch):
  """Added to in place, used twice, scaled by something that has a gradient itself; a second derivative is refused."""
  from t5x_b200.ops import native
  monkeypatch.setenv("T5X_B200_HOST_OPS", host)
  monkeypatch.setattr(native, "_host", None)
  d = data(4, 6, 700, torch.float32, 5)
  x = d["x"].clone().requires_grad_()
  base = torch.autograd.grad(call(kind, x, d, 2.0)[0], x)[0]
  scale = torch.tensor(3.0, device="cuda", requires_grad=True)
  out = call(kind, x, d, 2.0)
  value = float(out[0])
  loss = out[0]
  loss += 1.0
  gx, gs = torch.autograd.grad(loss * scale + 0.5 * loss, (x, scale))
  # (two products of 32 bits a value: 2^-23)
  assert torch.allclose(gx, base * 3.5, rtol=2 ** -22, atol=0) and float(gs) == pytest.approx(value + 1, rel=1e-6)
  assert not any(o.requires_grad for o in out[1:])
  gx = torch.autograd.grad(call(kind, x, d, 2.0)[0] * scale, x, create_graph=True)[0]
  with pytest.raises(RuntimeError, match="twice"):
    gx.sum().backward()


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_frozen_logits_and_inputs_with_gradients(kind):
  """Without a gradient of the logits no graph is built, and inputs beside them get none."""
  d = data(2, 5, 1500, torch.bfloat16, 6)
  out = call(kind, d["x"], d, None)
  assert not any(o.requires_grad for o in out)
  e = dict(d, **{k: d[k].clone().requires_grad_() for k in ("w", "r", "old")})
  assert not any(o.requires_grad for o in call(kind, d["x"], e, None))
  x = d["x"].clone().requires_grad_()
  got = torch.autograd.grad(call(kind, x, e, None)[0], [x, e["w"]], allow_unused=True)
  assert got[1] is None and torch.equal(got[0], torch.autograd.grad(call(kind, x, d, None)[0], x)[0])


def test_inference_mode():
  d = data(2, 4, 2000, torch.bfloat16, 7)
  want = call("policy", d["x"], d, None)
  with torch.inference_mode():
    got = call("policy", d["x"], d, None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.isfinite(call("preference", d["x"].clone(), d, None)[0])


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("dtype, vocab", [(torch.float32, 1800), (torch.bfloat16, 3501), (torch.float32, 1537),
                                          (torch.bfloat16, 4096), (torch.float32, 2049)])
def test_many_rows_of_some_kilobytes(kind, dtype, vocab):
  """More rows than run at once, about the sizes at which a row passes from a warp to the smallest blocks."""
  d = data(20, 150, vocab, dtype, seed=vocab)
  x = d["x"].requires_grad_()
  out = call(kind, x, d, 7.0)
  check(kind, out, torch.autograd.grad(out[0], x)[0], d, 7.0)


@pytest.mark.parametrize("vocab", [40000, 65537, 140001])
def test_rows_of_several_blocks_between_masked_ones(vocab):
  """Blocks that share a row do not meet at rows of weight 0: most rows here, so that a block may run ahead by several."""
  d = data(12, 60, vocab, torch.float32, seed=vocab, hidden=0.8)
  x = d["x"].requires_grad_()
  first = None
  for _ in range(10):
    out = call("policy", x, d, 7.0)
    grad = torch.autograd.grad(out[0], x)[0]
    if first is None:
      first = out, grad
      check("policy", out, grad, d, 7.0)
    assert torch.equal(grad, first[1]) and all(torch.equal(a, b) for a, b in zip(out, first[0]))
