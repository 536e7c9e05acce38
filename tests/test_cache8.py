"""Decoding in 8 bits as tensor operations (what runs on the CPU and states what the kernels compute): against loops in 64
bits, at the borders of blocks, rows and masks; refusals."""
import math

import pytest
import torch

from t5x_b200.ops import cache8
from t5x_b200.ops import functional as F


# ---- the definitions, a token at a time, in 64 bits --------------------------------------------------------------------
def code(x, most):
  return round(127 * x / most) if most > 0 and math.isfinite(most) else 0


def append_oracle(cache, name, x, starts, counts):
  """x [B, L, H, D] into copies of (codes, absmax), block by block."""
  codes, most = cache["cached_" + name].cpu().clone(), cache[name + "_absmax"].cpu().double().clone()
  b, h, slots, dim = codes.shape
  block = slots // most.shape[2]
  x = x.cpu().double()
  for i in range(b):
    start, stop = starts[i], min(starts[i] + counts[i], slots)
    for k in range(start // block, -(-stop // block) if stop > start else 0):
      lo, hi = max(start, k * block), min(stop, (k + 1) * block)
      for j in range(h):
        new = x[i, lo - start:hi - start, j]
        old = most[i, j, k].item() if lo > k * block else 0.0
        big = new.abs().max().item()
        a = big if math.isnan(big) or math.isnan(old) else max(old, big)
        a = math.nan if math.isnan(old) else a
        if a != old and lo > k * block:
          old_codes = codes[i, j, k * block:lo].double()
          again = torch.round(old_codes * old / a) if math.isfinite(a) else torch.zeros_like(old_codes)
          codes[i, j, k * block:lo] = torch.nan_to_num(again).to(torch.int8)
        fresh = torch.round(127 * new / a) if a > 0 and math.isfinite(a) else torch.zeros_like(new)
        codes[i, j, lo:hi] = torch.nan_to_num(fresh).to(torch.int8)
        most[i, j, k] = a
  return codes, most.float()


def bucket(d, num, far):
  d = max(d, 0)
  if d < num // 2:
    return d
  return min(num - 1, num // 2 + int(math.log(d / (num // 2)) / math.log(far / (num // 2)) * (num - num // 2) + 1e-6))


def attention_oracle(query, cache, starts, appended, table=None, num=32, far=128, mask=None, causal=True, scale=1.0):
  """(out, sum of p |v|, largest sum of |q| |k| and bias, weight by slot), all in 64 bits."""
  q = query.detach().cpu().double()
  codes = {n: cache["cached_" + n].cpu().double() for n in ("key", "value")}
  most = {n: cache[n + "_absmax"].cpu().double() for n in ("key", "value")}
  b, h, slots, dim = codes["key"].shape
  block = slots // most["key"].shape[2]
  count, group = q.shape[1], q.shape[2] // h
  out, size = torch.zeros_like(q), torch.zeros_like(q)
  weight, high = torch.zeros(b, h, slots, dtype=torch.float64), 0.0
  for i in range(b):
    end = min(starts[i] + appended, slots)
    for j in range(h):
      kv = {n: codes[n][i, j] * (most[n][i, j].repeat_interleave(block) / 127)[:, None] for n in codes}
      for l in range(count):
        own = starts[i] + appended - count + l
        seen = [s for s in range(end) if (not causal or s <= own) and
                (mask is None or (s < mask.shape[1] and bool(mask[i, s])))]
        if not seen:
          continue
        at = torch.tensor(seen)
        for g in range(group):
          x = q[i, l, j * group + g]
          s = scale * (kv["key"][at] @ x)
          size_s = abs(scale) * (kv["key"][at].abs() @ x.abs())
          if table is not None:
            place = cache["token_position"][i, j].cpu()[at].tolist() if "token_position" in cache else seen
            mine = own + (int(cache["dropped"][i]) if "token_position" in cache else 0)
            bias = torch.stack([table[j * group + g].cpu().double()[bucket(mine - p, num, far)] for p in place])
            s, size_s = s + bias, size_s + bias.abs()
          p = torch.softmax(s, 0)
          out[i, l, j * group + g] = p @ kv["value"][at]
          size[i, l, j * group + g] = p @ kv["value"][at].abs()
          weight[i, j, at] += p
          fine = size_s[torch.isfinite(size_s)]
          high = max(high, fine.max().item() if fine.numel() else 0.0)
  return out, size, high, weight


def within(got, want, size, high, dim, tokens):
  """Whether |got - want| is within half a step of the result's type, the roundings of probabilities and of scores.

  A score is a sum of `dim` products in 32 bits of a query that is held to 22 bits: off by (dim + 16) 2^-24 + 2^-21 of the
  sum of their magnitudes at most, and a probability by twice that, relatively. In 16-bit types a probability is rounded
  to 11 bits (2^-11 and its part below the rounding: 2^-10 with the sum of them that divides); in 32 bits it has 22. The
  sum over the tokens is in 32 bits."""
  eps = torch.finfo(got.dtype).eps / 2
  each = 2 * ((dim + 16) * 2.0 ** -24 + 2.0 ** -21) * high + (tokens + 64) * 2.0 ** -24
  each += 2.0 ** -10 if got.dtype != torch.float32 else 2.0 ** -20
  off = (got.cpu().double() - want).abs() - eps * want.abs() - each * size
  return bool((off <= torch.finfo(got.dtype).tiny).all())


def make(b, h, slots, dim, block, starts, seed=0, weights=False, positions=False, device="cpu", scalar=False):
  gen = torch.Generator().manual_seed(seed)
  cache = cache8.init_cache(b, slots, h, dim, device, block=block, weights=weights, positions=positions)
  for n in ("key", "value"):
    cache["cached_" + n].copy_(torch.randint(-127, 128, cache["cached_" + n].shape, generator=gen))
    cache[n + "_absmax"].copy_((1 + 2 * torch.rand(cache[n + "_absmax"].shape, generator=gen)).bfloat16())
  cache["cache_index"].copy_(torch.tensor(starts))
  if scalar:
    cache["cache_index"] = cache["cache_index"][0].clone()
  if weights:
    cache["token_weight"].copy_(torch.rand(cache["token_weight"].shape, generator=gen))
  if positions:
    cache["dropped"].copy_(torch.randint(0, 200, (b,), generator=gen))
    gaps = torch.randint(0, 5, cache["token_position"].shape, generator=gen).cumsum(2)
    at = torch.arange(cache["cached_key"].shape[2])
    cache["token_position"].copy_(torch.minimum(at + gaps, at + cache["dropped"].cpu()[:, None, None]))
  return cache


def tokens(b, count, h, dim, seed=1, dtype=torch.float32):
  gen = torch.Generator().manual_seed(seed)
  return [(torch.randn(b, count, h, dim, generator=gen) * m).to(dtype) for m in (1.5, 0.7)]


CASES = [
    # b, heads, group, dim, slots, block, starts, count, options
    dict(b=3, h=2, group=1, dim=64, slots=64, block=16, starts=[0, 15, 40], count=1),
    dict(b=2, h=1, group=2, dim=128, slots=96, block=32, starts=[31, 33], count=1, bias=True),
    dict(b=3, h=2, group=3, dim=64, slots=128, block=64, starts=[1, 64, 127], count=1, weights=True, positions=True, bias=True),
    dict(b=2, h=2, group=1, dim=64, slots=128, block=16, starts=[3, 60], count=21, bias=True, weights=True),
    dict(b=2, h=1, group=4, dim=64, slots=64, block=16, starts=[10, 60], count=9),  # (the second runs over the end)
    dict(b=2, h=2, group=1, dim=64, slots=80, block=16, starts=[80, 37], count=3, cross=True, mask=True, weights=True),
    dict(b=2, h=1, group=1, dim=64, slots=64, block=32, starts=[5, 50], count=6, own=True, weights=True),
    dict(b=2, h=1, group=1, dim=64, slots=64, block=32, starts=[7, 7], count=1, scalar=True, bias=True, scale=0.125),
    dict(b=1, h=1, group=9, dim=128, slots=16, block=16, starts=[0], count=1),
    dict(b=2, h=1, group=1, dim=64, slots=64, block=64, starts=[40, 64], count=2, mask=True),
]


def inputs(c, device="cpu", dtype=torch.float32, seed=0):
  cache = make(c["b"], c["h"], c["slots"], c["dim"], c["block"], c["starts"], seed, c.get("weights", False),
               c.get("positions", False), device, c.get("scalar", False))
  gen = torch.Generator().manual_seed(seed + 7)
  heads = c["h"] * c["group"]
  query = (torch.randn(c["b"], c["count"], heads, c["dim"], generator=gen) * 0.2).to(dtype).to(device)
  key, value = [None, None] if c.get("cross") or c.get("own") else \
      [t.to(device) for t in tokens(c["b"], c["count"], c["h"], c["dim"], seed + 1, dtype)]
  table = torch.randn(heads, 32, generator=gen).to(device) if c.get("bias") else None
  mask = None
  if c.get("mask"):
    mask = torch.rand(c["b"], c["slots"] - 5, generator=gen) > 0.4
    mask[-1] = False  # a row that sees nothing
    mask = mask.to(device)
  kw = dict(bias_table=table, key_mask=mask, causal=not c.get("cross"), scale=c.get("scale", 1.0))
  return cache, query, key, value, kw


def check_attention(c, device="cpu", dtype=torch.float32, seed=0):
  cache, query, key, value, kw = inputs(c, device, dtype, seed)
  before = {k: v.cpu().clone() for k, v in cache.items()}
  out = cache8.attention(query, cache, key, value, **kw)
  assert out.shape == query.shape and out.dtype == dtype
  appended = 0 if key is None else c["count"]
  for n, x in (("key", key), ("value", value)):
    if x is not None:
      codes, most = append_oracle(before, n, x, c["starts"], [c["count"]] * c["b"])
      assert torch.equal(cache["cached_" + n].cpu(), codes) and torch.equal(cache[n + "_absmax"].cpu(), most)
  assert torch.equal(cache["cache_index"].cpu(), before["cache_index"])
  for i, s in enumerate(c["starts"]):
    new = slice(s, min(s + appended, c["slots"]))
    if c.get("positions"):
      before["token_position"][i, :, new] = torch.arange(new.start, new.stop, dtype=torch.int32) + before["dropped"][i]
    if c.get("weights"):
      before["token_weight"][i, :, new] = 0
  if c.get("positions"):
    assert torch.equal(cache["token_position"].cpu(), before["token_position"])
  want, size, high, weight = attention_oracle(query, cache, c["starts"], appended, kw["bias_table"], mask=kw["key_mask"],
                                              causal=kw["causal"], scale=kw["scale"])
  assert within(out, want, size, high, c["dim"], c["slots"])
  if c.get("weights"):
    # as in `within`, without the rounding of the probabilities: the sums are of the unrounded ones
    each = 2 * ((c["dim"] + 16) * 2.0 ** -24 + 2.0 ** -21) * high + (c["slots"] + 64) * 2.0 ** -24 + 2.0 ** -20
    off = (cache["token_weight"].cpu().double() - before["token_weight"].double() - weight).abs()
    assert bool((off <= each * weight + 2.0 ** -22 * before["token_weight"].double() + 1e-30).all())
  return out, cache


@pytest.mark.parametrize("c", CASES, ids=range(len(CASES)))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention(c, dtype):
  check_attention(c, "cpu", dtype)


@pytest.mark.parametrize("lengths", [None, [0, 1, 33]])
def test_append_and_values(lengths):
  cache = make(3, 2, 64, 64, 16, [0, 17, 30])
  before = {k: v.clone() for k, v in cache.items()}
  key, value = tokens(3, 33, 2, 64)
  cache8.append_(cache, key, value, None if lengths is None else torch.tensor(lengths))
  for n, x in (("key", key), ("value", value)):
    codes, most = append_oracle(before, n, x, [0, 17, 30], lengths or [33] * 3)
    assert torch.equal(cache["cached_" + n], codes) and torch.equal(cache[n + "_absmax"], most)
  if lengths is None:  # half a step of the block's scale, and another for codes that were rounded again
    held = cache["cached_key"][0, :, :33].float() * cache["key_absmax"][0].repeat_interleave(16, 1)[:, :33, None] / 127
    off = (held - key[0].transpose(0, 1)).abs()
    assert bool((off <= cache["key_absmax"][0].repeat_interleave(16, 1)[:, :33, None] / 127 * 0.5001).all())


def test_token_by_token_is_a_repeat_of_the_same_blocks():
  """One token at a time gives the scales of all at once, and appending the same tokens again changes nothing."""
  key, value = tokens(2, 40, 1, 64)
  whole, single = (cache8.init_cache(2, 64, 1, 64, block=16) for _ in range(2))
  cache8.append_(whole, key, value)
  for i in range(40):
    cache8.append_(single, key[:, i:i + 1], value[:, i:i + 1])
    again = single["cached_key"].clone()
    cache8.append_(single, key[:, i:i + 1], value[:, i:i + 1])
    assert torch.equal(again, single["cached_key"])
    single["cache_index"] += 1
  assert torch.equal(whole["key_absmax"], single["key_absmax"])
  # (each time that a block's scale grows its codes are off by another half step)
  assert (whole["cached_key"].int() - single["cached_key"].int()).abs().max() <= 8


def check_zeros_into_a_used_block(device="cpu"):
  """A block that begins anew does not keep the scale that its slots had before."""
  cache = make(2, 1, 32, 64, 16, [16, 0], device=device)
  zeros = torch.zeros(2, 1, 1, 64, device=device)
  out = cache8.attention(zeros, cache, zeros, zeros)
  assert cache["key_absmax"][0, 0, 1] == 0 and cache["value_absmax"][1, 0, 0] == 0 and (cache["cached_key"][0, 0, 16] == 0).all()
  assert (out[1] == 0).all() and not out.isnan().any()


def test_zeros_into_a_used_block():
  check_zeros_into_a_used_block()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(bad):
  c = dict(b=1, h=1, group=1, dim=64, slots=64, block=16, starts=[20], count=1)
  cache, query, key, value, kw = inputs(c)
  value[0, 0, 0, 3] = bad
  hide = torch.ones(1, 64, dtype=torch.bool)
  hide[0, 16:32] = False  # the block that gets it
  want = cache8.attention(query, {k: v.clone() for k, v in cache.items()}, *tokens(1, 1, 1, 64), key_mask=hide, **{
      k: v for k, v in kw.items() if k != "key_mask"})
  out = cache8.attention(query, cache, key, value, key_mask=hide)
  assert torch.equal(out, want)
  assert cache8.attention(query, cache, key, value).isnan().all()
  assert (cache["cached_value"][0, 0, 16:21] == 0).all()


@pytest.mark.parametrize("most", [1e-44, 1e-38, 1e-30, 3e38])
def test_blocks_of_the_smallest_and_largest_values(most):
  cache = cache8.init_cache(1, 16, 1, 64, block=16)
  key = torch.linspace(-1, 1, 64).view(1, 1, 1, 64) * most
  cache8.append_(cache, key, key)
  big = key.abs().max().item()
  assert cache["key_absmax"].item() == big
  assert cache["cached_key"][0, 0, 0].tolist() == [round(127 * x / big) for x in key.flatten().tolist()]


# ---- eviction ----------------------------------------------------------------------------------------------------------
def evict_oracle(cache, keep, recent, into):
  b, h, slots, dim = cache["cached_key"].shape
  block, to_block = slots // cache["key_absmax"].shape[2], into["cached_key"].shape[2] // into["key_absmax"].shape[2]
  out = {k: v.cpu().clone() for k, v in into.items()}
  kept = torch.full((b, h, keep), -1, dtype=torch.int32)
  for i in range(b):
    index = int(cache["cache_index"].expand(b)[i])
    held = min(index, slots)
    for j in range(h):
      w = cache["token_weight"][i, j].tolist()
      old = max(0, held - recent)
      order = sorted(range(old), key=lambda s: (0 if math.isnan(w[s]) else 1, -w[s] if w[s] == w[s] else 0, s))
      stay = sorted(order[:keep - (held - old)] + list(range(old, held))) if held > keep else list(range(held))
      kept[i, j, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
      for n, s in enumerate(stay):
        out["token_weight"][i, j, n] = cache["token_weight"][i, j, s]
        out["token_position"][i, j, n] = cache["token_position"][i, j, s] if "token_position" in cache else s
      for name in ("key", "value"):
        for k in range(0, len(stay), to_block):
          part = stay[k:k + to_block]
          a = [cache[name + "_absmax"][i, j, s // block].double().item() for s in part]
          big = max(a)
          out[name + "_absmax"][i, j, k // to_block] = big
          for n, (s, x) in enumerate(zip(part, a)):
            c = cache["cached_" + name][i, j, s].cpu().double()
            out["cached_" + name][i, j, k + n] = (torch.round(c * x / big) if x != big else c).to(torch.int8)
    out["cache_index"][i] = min(held, keep)
    before = int(cache["dropped"][i]) if "token_position" in cache else 0
    out["dropped"][i] = before + index - min(held, keep)
  return kept, out


EVICT = [
    dict(b=3, h=2, dim=64, slots=64, block=16, starts=[64, 33, 10], keep=17, recent=5, positions=True),
    dict(b=2, h=1, dim=128, slots=256, block=32, starts=[200, 256], keep=100, recent=100),
    dict(b=2, h=3, dim=64, slots=128, block=64, starts=[90, 128], keep=33, recent=0, to_block=16),
    dict(b=2, h=1, dim=64, slots=128, block=16, starts=[0, 1], keep=1, recent=0, positions=True),
    dict(b=1, h=1, dim=64, slots=64, block=16, starts=[70], keep=1, recent=1),  # (an index behind the end)
    dict(b=2, h=2, dim=64, slots=64, block=16, starts=[60, 50], keep=64, recent=3),
    dict(b=1, h=2, dim=64, slots=2304, block=128, starts=[2300], keep=1029, recent=7, to_block=32, positions=True),
]


def check_evict(c, device="cpu", special=False):
  cache = make(c["b"], c["h"], c["slots"], c["dim"], c["block"], c["starts"], 3, True, c.get("positions", False), device)
  w = cache["token_weight"]
  w.copy_((w * 8).floor() / 8)  # many ties
  if special:
    w[:, :, ::7], w[:, :, 1::7], w[:, :, 2::7], w[:, :, 3::7] = math.nan, math.inf, -math.inf, -0.0
    w[:, :, 4::7], w[:, :, 5::7], w[:, :, 6::7] = 0.0, 1e-41, -1e-41
  before = {k: v.clone() for k, v in cache.items()}
  into = make(c["b"], c["h"], -(-c["keep"] // c.get("to_block", c["block"])) * c.get("to_block", c["block"]), c["dim"],
              c.get("to_block", c["block"]), [0] * c["b"], 4, True, True, device)
  kept_want, want = evict_oracle({k: v.cpu() for k, v in cache.items()}, c["keep"], c["recent"], into)
  out, kept = cache8.evict(cache, c["keep"], recent=c["recent"], out=into)
  assert out is into and torch.equal(kept.cpu(), kept_want)
  for n, t in want.items():
    assert torch.equal(out[n].cpu().nan_to_num(7.0) if t.is_floating_point() else out[n].cpu(),
                       t.nan_to_num(7.0) if t.is_floating_point() else t), n
  assert all(torch.equal(cache[n].nan_to_num(7.0) if cache[n].is_floating_point() else cache[n],
                         t.nan_to_num(7.0) if t.is_floating_point() else t) for n, t in before.items())


@pytest.mark.parametrize("c", EVICT, ids=range(len(EVICT)))
@pytest.mark.parametrize("special", [False, True])
def test_evict(c, special):
  check_evict(c, special=special)


def test_evict_into_a_new_cache():
  cache = make(2, 1, 64, 64, 16, [64, 30], weights=True)
  out, kept = cache8.evict(cache, 40, recent=8)
  assert out["cached_key"].shape == cache["cached_key"].shape and out["cache_index"].tolist() == [40, 30]
  assert out["dropped"].tolist() == [24, 0] and kept.shape == (2, 1, 40)
  assert (out["cached_key"][1, :, 30:] == 0).all()


# ---- products ----------------------------------------------------------------------------------------------------------
def linear_oracle(x, weight, residual=None):
  """(y in 64 bits, what 32 bits may be off by: the products with the scales, and the residual's sum)."""
  x = x.detach().cpu().double()
  codes, absmax, k = weight
  rows = []
  for r in x:
    most = r.abs().max().item()
    cx = torch.tensor([float(code(v, most)) for v in r.tolist()], dtype=torch.float64)
    rows.append(torch.mv(codes[:, :k].cpu().double(), cx) * most / 127 * absmax.cpu().double() / 127)
  y = torch.stack(rows) if rows else torch.zeros(0, codes.shape[0], dtype=torch.float64)
  size = y.abs()
  if residual is not None:
    y, size = y + residual.cpu().double(), size + residual.cpu().double().abs()
  return y, size * 2.0 ** -21  # (eight roundings of 2^-24)


def check_linear(rows, k, n, dtype, residual, device="cpu", seed=0):
  gen = torch.Generator().manual_seed(seed)
  w = torch.randn(k, n, generator=gen) * 0.1
  x = (torch.randn(rows, k, generator=gen) * torch.exp(2 * torch.randn(rows, 1, generator=gen))).to(dtype)
  if rows > 1:
    x[rows // 2] = 0
  r = torch.randn(rows, n, generator=gen).to(dtype) if residual else None
  weight = F.quantize_weight(w.to(device))
  want_codes = torch.tensor([[code(v, c.abs().max().item()) for v in c.tolist()] for c in w.t()])
  assert torch.equal(weight.codes[:, :k].cpu().long(), want_codes) and (weight.codes[:, k:] == 0).all()
  assert torch.equal(weight.absmax.cpu(), w.abs().amax(0))
  y = F.linear8(x.to(device), weight, None if r is None else r.to(device))
  assert y.dtype == dtype and y.shape == (rows, n)
  want, size = linear_oracle(x, weight, r)
  info = torch.finfo(dtype)
  off = (y.cpu().double() - want).abs() - info.eps / 2 * want.abs()
  # (results below the smallest normal number are a whole number of its steps: half a step is smallest * eps / 2)
  assert bool((off <= size * (1 + info.eps) + info.smallest_normal * info.eps / 2).all())


@pytest.mark.parametrize("rows,k,n", [(1, 16, 8), (3, 17, 5), (5, 1, 3), (0, 8, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear8(rows, k, n, dtype):
  check_linear(rows, k, n, dtype, rows == 3)


def test_linear8_keeps_leading_dims_and_nan_rows():
  weight = F.quantize_weight(torch.randn(8, 2, 3))
  x = torch.randn(2, 3, 8)
  x[0, 1, 4] = math.inf
  y = F.linear8(x, weight)
  assert y.shape == (2, 3, 6) and y[0, 1].isnan().all() and not y[0, 0].isnan().any()


# ---- refusals ----------------------------------------------------------------------------------------------------------
def test_refusals():
  cache = make(2, 2, 64, 64, 16, [3, 4], weights=True)
  q = torch.randn(2, 1, 4, 64)
  k = torch.randn(2, 1, 2, 64)
  three = make(3, 2, 64, 64, 16, [3, 4, 5], weights=True, positions=True)
  bad = [
      lambda: cache8.init_cache(1, 8, 1, 64, block=24),
      lambda: cache8.init_cache(1, 0, 1, 64),
      lambda: cache8.attention(q[:1], cache, k, k),
      lambda: cache8.attention(q[:, :, :3], cache, k, k),
      lambda: cache8.attention(q[..., :32], cache, k, k),
      lambda: cache8.attention(q, cache, k),
      lambda: cache8.attention(q, cache, k.double(), k.double()),
      lambda: cache8.attention(q, cache, k.expand(2, 2, 2, 64), k.expand(2, 2, 2, 64)),
      lambda: cache8.attention(q, cache, k, k[:, :, :1]),
      lambda: cache8.attention(q, cache, k, k, bias_table=torch.zeros(3, 32)),
      lambda: cache8.attention(q, cache, k, k, bias_table=torch.zeros(4, 31)),
      lambda: cache8.attention(q, cache, k, k, bias_table=torch.zeros(4, 32), max_distance=16),
      lambda: cache8.attention(q, cache, k, k, key_mask=torch.ones(2, 65, dtype=torch.bool)),
      lambda: cache8.attention(q, cache, k, k, key_mask=torch.ones(2, 1, 64, dtype=torch.bool)),
      lambda: cache8.attention(q.clone().requires_grad_(), cache, k, k),
      lambda: cache8.attention(q.long(), cache, k, k),
      lambda: cache8.append_(cache, k, k, torch.ones(3, dtype=torch.int32)),
      lambda: cache8.append_(cache, k, k, torch.ones(2)),
      lambda: cache8.append_(cache, k[:, :0], k[:, :0]),
      lambda: cache8.append_(cache | {"key_absmax": cache["key_absmax"][:, :, :3]}, k, k),
      lambda: cache8.append_(cache | {"cached_value": cache["cached_value"].transpose(1, 2)}, k, k),
      lambda: cache8.append_(cache | {"cache_index": cache["cache_index"].long()}, k, k),
      lambda: cache8.append_({"cached_key": cache["cached_key"]}, k, k),
      lambda: cache8.append_(cache | {"token_position": torch.zeros(2, 2, 64, dtype=torch.int32)}, k, k),
      lambda: cache8.evict(cache, 0),
      lambda: cache8.evict(cache, 8, recent=9),
      lambda: cache8.evict(cache, 65),
      lambda: cache8.evict(cache, 8, out=cache),
      lambda: cache8.evict(cache, 8, out=make(2, 2, 64, 64, 16, [0, 0], weights=True)),
      lambda: cache8.evict({n: t[:2] for n, t in three.items()}, 8, out={n: t[1:] for n, t in three.items()}),
      lambda: cache8.evict(make(2, 2, 64, 64, 16, [3, 4]), 8),
      lambda: cache8.evict(cache, 33, out=make(2, 2, 32, 64, 16, [0, 0], weights=True, positions=True)),
      lambda: F.quantize_weight(torch.ones(4, 4, dtype=torch.long)),
      lambda: F.linear8(torch.randn(2, 7), F.quantize_weight(torch.randn(8, 4))),
      lambda: F.linear8(torch.randn(2, 8).requires_grad_(), F.quantize_weight(torch.randn(8, 4))),
      lambda: F.linear8(torch.randn(2, 8), F.quantize_weight(torch.randn(8, 4)), torch.randn(2, 5)),
      lambda: F.linear8(torch.randn(2, 8), F.quantize_weight(torch.randn(8, 4)), torch.randn(2, 4).double()),
  ]
  before = {n: t.clone() for n, t in cache.items()}
  for i, call in enumerate(bad):
    with pytest.raises(ValueError):
      call()
      pytest.fail(f"call {i} was not refused")
  assert all(torch.equal(cache[n], t) for n, t in before.items())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("name", ["token_weight", "token_position", "dropped"])
def test_entries_that_are_no_tensors(device, name):
  """They would go without their weights or positions."""
  whole = make(2, 2, 64, 64, 16, [3, 4], weights=True, positions=True, device=device)
  other = make(2, 2, 64, 64, 16, [0, 0], weights=True, positions=True, device=device)
  q, k = torch.randn(2, 1, 4, 64, device=device), torch.randn(2, 1, 2, 64, device=device)
  for strange in (None, whole[name].cpu().numpy(), whole[name].tolist()):
    cache = whole | {name: strange}
    for call in (lambda: cache8.attention(q, cache, k, k), lambda: cache8.append_(cache, k, k),  # noqa: B023
                 lambda: cache8.evict(cache, 2, out=other), lambda: cache8.evict(whole, 2, out=other | {name: strange})):  # noqa: B023
      with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refusals_are_the_same_on_every_device(device):
  cache = make(2, 2, 64, 64, 16, [3, 4], weights=True, device=device)
  one = make(1, 1, 64, 64, 16, [3], weights=True, device=device)
  into = make(1, 1, 64, 64, 16, [0], weights=True, positions=True, device=device)
  q, k = torch.randn(2, 1, 4, 64, device=device), torch.randn(2, 1, 2, 64, device=device)
  long = cache8.init_cache(1, 1 << 17, 1, 64, device, weights=True)
  for call in (lambda: cache8.attention(q, cache, k, k, bias_table=torch.zeros(4, 1, device=device), num_buckets=1),
               lambda: cache8.attention(q, cache, k, k, bias_table=torch.zeros(4, 0, device=device), num_buckets=0),
               lambda: cache8.attention(q, cache, k, k, bias_table=torch.zeros((), device=device)),
               # 2^31 scores whose weight is added up
               lambda: cache8.attention(torch.zeros(1, 1, 1 << 14, 64, device=device), long),
               lambda: cache8.evict(one, 2, out=into | {"cache_index": into["cache_index"][0]})):
    with pytest.raises(ValueError):
      call()
