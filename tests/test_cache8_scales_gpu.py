"""Attention over a cache in 8 bits whose blocks have scales far apart, and whose rows see little of a block: what is hidden
changes no bit, a block that is not finite is NaN to all that see it, and few tokens of much weight do not cost the others theirs."""
import math

import pytest
import torch

import test_cache8 as plain
from t5x_b200.ops import cache8
from t5x_b200.ops import native

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def attend(*args, **kw):
  before = native.launch_count()
  out = cache8.attention(*args, **kw)
  assert native.launch_count() > before
  return out


# (dim, heads that share keys, queries, tokens held, slots): rows of up to four, of five to eight, of a tile, of two, in pieces
SIGHTS = [(64, 1, 4, 22, 64), (64, 1, 6, 22, 64), (64, 8, 1, 19, 64), (128, 2, 3, 22, 64), (64, 3, 6, 22, 64), (64, 40, 6, 22, 64),
          (128, 40, 6, 22, 96), (64, 1, 6, 22, 2112), (64, 7, 1, 19, 2112), (128, 1, 6, 22, 2112), (64, 30, 6, 22, 2112)]


@pytest.mark.parametrize("big", [2.0 ** 16, 2.0 ** 29, 3e38, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group,count,held,slots", SIGHTS)
def test_a_block_of_which_a_row_sees_nothing(dim, group, count, held, slots, dtype, big):
  """The mask hides a block's first tokens and shows later ones, which the causal limit hides from the first queries (or which
  are not held): their results have the same bits whatever the block's largest value."""
  c = dict(b=1, h=1, group=group, dim=dim, slots=slots, block=16, starts=[held], count=count, own=True)
  cache, query, _, _, _ = plain.inputs(c, "cuda", dtype)
  shown = torch.ones(1, slots, dtype=torch.bool, device="cuda")
  shown[0, 16:20] = False
  blind = max(0, 20 - (held - count))  # queries that see nothing from slot 16 on
  assert 0 < blind <= 4
  cache["value_absmax"].fill_(1.0)
  want = attend(query, cache, key_mask=shown)[:, :blind]
  cache["value_absmax"][0, 0, 1] = big
  if not math.isfinite(big):
    cache["cached_value"][0, 0, 16:32] = 0  # as such a block is held
  got = attend(query, cache, key_mask=shown)[:, :blind]
  assert want.isfinite().all() and (want != 0).any() and torch.equal(got, want)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group,count,slots", [(64, 4, 1, 64), (64, 8, 1, 64), (128, 4, 1, 64), (128, 8, 1, 2112), (64, 2, 2, 2112),
                                                   (64, 20, 1, 64), (128, 50, 4, 64)])
def test_a_key_block_that_is_not_finite(dim, group, count, slots, dtype, bad):
  """NaN for each of a thousand queries that see it, nothing to those that a mask hides it from."""
  rows = -(-1000 // (group * count))
  gen = torch.Generator("cuda").manual_seed(0)
  cache = cache8.init_cache(rows, slots, 1, dim, "cuda", block=16)
  for n in ("key", "value"):
    cache["cached_" + n].copy_(torch.randint(-127, 128, cache["cached_" + n].shape, generator=gen, device="cuda", dtype=torch.int8))
    cache[n + "_absmax"].fill_(1.0)
  cache["cache_index"].fill_(40)
  query = torch.randn(rows, count, group, dim, generator=gen, device="cuda").to(dtype)
  shown = torch.ones(rows, slots, dtype=torch.bool, device="cuda")
  shown[:, 16:32] = False
  want = attend(query, cache, key_mask=shown)
  cache["cached_key"][:, :, 16:32] = 0
  cache["key_absmax"][:, :, 1] = bad
  assert want.isfinite().all() and torch.equal(attend(query, cache, key_mask=shown), want)
  assert attend(query, cache).isnan().all()


def scene(dim, group, count, tokens, dtype, nats, scales, at=37):
  """A cache of `tokens` tokens whose score is 0.3, but for one of score `nats` at slot `at`; scales: largest values of the
  value blocks, of the one's and of the others. (The query has one channel: scores have few roundings.)"""
  gen = torch.Generator("cuda").manual_seed(3)
  cache = cache8.init_cache(1, tokens, 1, dim, "cuda", block=16)
  cache["cached_value"].copy_(torch.randint(-127, 128, cache["cached_value"].shape, generator=gen, device="cuda", dtype=torch.int8))
  cache["value_absmax"].fill_(scales[1])
  cache["value_absmax"][0, 0, at // 16] = scales[0]
  mine = cache["cached_value"][0, 0, at].clone()
  cache["cached_value"][0, 0, at // 16 * 16:at // 16 * 16 + 16] = 0  # (the block's other tokens have values of 0)
  cache["cached_value"][0, 0, at] = mine
  cache["key_absmax"].fill_(0.3)
  cache["cached_key"][..., 0] = 127
  cache["key_absmax"][0, 0, at // 16] = abs(nats)
  cache["cached_key"][0, 0, at // 16 * 16:at // 16 * 16 + 16, 0] = round(127 * 0.3 / abs(nats))
  cache["cached_key"][0, 0, at, 0] = 127 if nats > 0 else -127
  cache["cache_index"].fill_(tokens)
  query = torch.zeros(1, count, group, dim, device="cuda", dtype=dtype)
  query[..., 0] = 1.0
  return query, cache


def check(query, cache, dtype):
  """Against 64 bits.

  Roundings: scores have about eight of 32 bits (scales, one product, the reference's subtraction), a probability has twice
  their sum and 2^-21 of its own; 16-bit types round it to 11 bits (2^-10 with the sum that divides). Sums of 16 tokens are
  added up in 32 bits, one after the other at most. What a probability times its block's largest value is off below fp16's
  normal numbers is half of 2^-24 (in 32 bits, with a second number at 2^-11, half of 2^-35) where the largest is 2^6 or more."""
  tokens, dim = cache["cached_key"].shape[2:]
  out = attend(query, cache, causal=False)
  most = {n: cache[n + "_absmax"][0, 0].double().repeat_interleave(16) for n in ("key", "value")}
  k, v = [cache["cached_" + n][0, 0].double() * most[n][:, None] / 127 for n in ("key", "value")]
  s = query[0].double().flatten(0, 1) @ k.t()
  p = torch.softmax(s, 1)
  want, size = p @ v, p @ v.abs()
  top = (p * most["value"]).amax(1, keepdim=True)
  wide = dtype == torch.float32
  each = 16 * 2.0 ** -24 * s.abs().max() + (tokens // 16 + 64) * 2.0 ** -24 + 2.0 ** -21 + (0 if wide else 2.0 ** -10)
  floor = tokens * top * (2.0 ** -42 if wide else 2.0 ** -31)
  off = (out[0].double().flatten(0, 1) - want).abs() - torch.finfo(dtype).eps / 2 * want.abs() - each * size - floor
  # (an output below the type's normal numbers is a whole number of its steps)
  assert bool((off <= torch.finfo(dtype).smallest_normal).all()), (off / (size + 1e-300)).max()


FORMS = [(64, 1, 1), (64, 6, 1), (128, 8, 1), (64, 20, 1), (128, 75, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group,count", FORMS)
@pytest.mark.parametrize("tokens", [1024, 8192])
@pytest.mark.parametrize("nats", [8.0, 10.0, 12.25, 15.0])
def test_one_token_far_above_the_others(dim, group, count, tokens, nats, dtype):
  for scales in ((1.0, 1.0), (1.0, 0.25), (1.0, 1 / 32), (1 / 32, 1.0), (1e-3, 1.0)):
    query, cache = scene(dim, group, count, tokens, dtype, nats, scales)
    check(query, cache, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group,count", FORMS)
@pytest.mark.parametrize("tokens", [1024, 8192])
@pytest.mark.parametrize("ratio", [4.0, 30.0, 1000.0, 30000.0, 2.0 ** 30, 1e30])
def test_a_block_far_larger_than_the_others(dim, group, count, tokens, ratio, dtype):
  """With little weight, and with next to none."""
  for nats in (-math.log(ratio), -math.log(ratio) - 8, -80.0):
    for at in (3, 517):
      # (fp16 has no results beyond 65504)
      query, cache = scene(dim, group, count, tokens, dtype, nats, (ratio, 1.0), at)
      check(query, cache, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,group,count", FORMS)
def test_blocks_of_the_largest_and_smallest_values(dim, group, count, dtype):
  """Values of 2^90 with next to no weight behind values of 2^-60, in tiles of one step and of several."""
  for at in (3, 20, 517):
    for scales in ((2.0 ** 90, 2.0 ** -60), (2.0 ** -60, 2.0 ** 60), (0.0, 1.0)):
      query, cache = scene(dim, group, count, 1024, dtype, -100.0 if scales[0] > 1 else 5.0, scales, at)
      check(query, cache, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,group,count", FORMS)
@pytest.mark.parametrize("tokens", [64, 4096])
@pytest.mark.parametrize("spread", [0, 4, 30])
def test_biases_of_the_lowest_value_over_blocks_of_any_scale(dim, group, count, tokens, spread, dtype):
  """All that a row sees has the lowest bias: its softmax is uniform, whatever the blocks' largest values are."""
  gen = torch.Generator("cuda").manual_seed(5)
  for size in (2.0 ** -60, 1e-6, 1e6, 2.0 ** 60):
    cache = cache8.init_cache(1, tokens, 1, dim, "cuda", block=16)
    cache["cached_value"].copy_(torch.randint(-127, 128, cache["cached_value"].shape, generator=gen, device="cuda", dtype=torch.int8))
    cache["cached_key"].copy_(torch.randint(-127, 128, cache["cached_key"].shape, generator=gen, device="cuda", dtype=torch.int8))
    cache["key_absmax"].fill_(1.0)
    down = torch.randint(-spread, 1, (tokens // 16,), generator=gen, device="cuda")
    most = torch.ldexp(torch.full_like(down, size, dtype=torch.float32), down)
    cache["value_absmax"][0, 0] = most
    cache["cache_index"].fill_(tokens)
    query = torch.randn(1, count, group, dim, generator=gen, device="cuda").to(dtype)
    out = attend(query, cache, bias_table=torch.full((group, 32), torch.finfo(torch.float32).min, device="cuda"), causal=False)
    v = cache["cached_value"][0, 0].double() * most.double().repeat_interleave(16)[:, None] / 127
    want, each = v.mean(0), v.abs().mean(0)
    # a probability is rounded once and in 32 bits; the largest term is that of the largest block
    floor = most.max().double() * (2.0 ** -42 if dtype == torch.float32 else 2.0 ** -31)
    bound = each * ((0 if dtype == torch.float32 else 2.0 ** -10) + (tokens // 16 + 64) * 2.0 ** -24 + 2.0 ** -21) + floor
    off = (out[0].double().flatten(0, 1) - want).abs() - torch.finfo(dtype).eps / 2 * want.abs()
    assert bool((off <= bound).all()), (size, (off / each).max())
