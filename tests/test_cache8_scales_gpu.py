"""Attention over a cache in 8 bits whose blocks have scales far apart, and whose rows see little of a block: what is hidden
changes no bit, a block that is not finite is NaN to all that see it."""
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
