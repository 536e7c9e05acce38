"""Kernels of decoding in 8 bits: against loops in 64 bits (test_cache8.py) at the borders of blocks, tiles, rows and masks;
strides, streams, captures; long caches against the statements in tensor operations."""
import math
import threading

import pytest
import torch

import test_cache8 as plain
from t5x_b200.ops import cache8
from t5x_b200.ops import functional as F
from t5x_b200.ops import native
from t5x_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]

MORE = [
    dict(b=2, h=2, group=5, dim=128, slots=128, block=16, starts=[0, 99], count=7, bias=True, weights=True, positions=True),
    dict(b=2, h=1, group=1, dim=64, slots=608, block=32, starts=[560, 13], count=40, bias=True, weights=True),
    dict(b=1, h=3, group=1, dim=128, slots=640, block=128, starts=[517], count=1, weights=True, mask=True),
    dict(b=1, h=1, group=40, dim=64, slots=528, block=16, starts=[511], count=1, bias=True),
    dict(b=2, h=1, group=1, dim=128, slots=64, block=64, starts=[63, 64], count=33, cross=True, weights=True),
    dict(b=2, h=2, group=2, dim=64, slots=1040, block=16, starts=[1000, 257], count=1, weights=True, positions=True, bias=True),
    dict(b=2, h=1, group=3, dim=128, slots=32, block=32, starts=[2, 30], count=5, own=True, weights=True),
]


def launches(call):
  before = native.launch_count()
  out = call()
  assert native.launch_count() > before
  return out


@pytest.mark.parametrize("c", plain.CASES + MORE, ids=range(len(plain.CASES + MORE)))
@pytest.mark.parametrize("dtype", TYPES)
def test_attention(c, dtype):
  launches(lambda: plain.check_attention(c, "cuda", dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 128)])
@pytest.mark.parametrize("lengths", [None, [0, 1, 33], [-4, 90, 2]])
def test_append(dtype, dim, block, lengths):
  cache = plain.make(3, 2, 128, dim, block, [0, 17, 120], device="cuda")
  before = {k: v.clone() for k, v in cache.items()}
  key, value = [t.cuda() for t in plain.tokens(3, 33, 2, dim, dtype=dtype)]
  given = None if lengths is None else torch.tensor(lengths).cuda()
  launches(lambda: cache8.append_(cache, key, value, given))
  for n, x in (("key", key), ("value", value)):
    codes, most = plain.append_oracle(before, n, x, [0, 17, 120], [min(max(v, 0), 33) for v in lengths or [33] * 3])
    assert torch.equal(cache["cached_" + n].cpu(), codes) and torch.equal(cache[n + "_absmax"].cpu(), most)


def test_zeros_into_a_used_block():
  plain.check_zeros_into_a_used_block("cuda")


def test_codes_at_every_border():
  """Values whose quotient lies on a border between two codes, or next to it, in 32 bits."""
  most = torch.tensor([1.0, 127.0, 2.5390625, 0.7071068286895752, 3.0e-39, 2.0e38])
  x = torch.zeros(6, 4096)
  for i, m in enumerate(most.tolist()):
    at = (torch.arange(-127, 127) + 0.5).double() * m / 127
    near = torch.stack([at.float(), torch.nextafter(at.float(), torch.tensor(math.inf)),
                        torch.nextafter(at.float(), torch.tensor(-math.inf))]).flatten()
    x[i, :near.numel()] = near.clamp(-m, m)
    x[i, -1] = m
  codes, absmax = native.quantize_rows(x.cuda(), 4096)
  want, size = ref.quantize_rows(x)
  assert torch.equal(codes.cpu(), want) and torch.equal(absmax.cpu(), size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_of_all_short_values(dtype):
  """Every positive value of a 16-bit type below each of many largest ones, and every code by many ratios of scales: where the
  quotient is on a border, and next to it."""
  bits = torch.arange(0x7f80 if dtype == torch.bfloat16 else 0x7c00, dtype=torch.int32)
  values = bits.to(torch.int16).view(dtype)
  one = torch.finfo(dtype).eps
  ends = torch.cat([1 + one * torch.arange(0, int(1 / one), 1 if dtype == torch.bfloat16 else 37), torch.tensor([2.0])]).to(dtype)
  near = values[(values.float() > 2.0 ** -9) & (values.float() <= 2)]
  x = torch.where(near[None] <= ends[:, None], near[None], torch.zeros((), dtype=dtype))
  x[:, -1] = ends
  codes, most = native.quantize_rows(x.cuda(), x.shape[1])
  assert torch.equal(most.cpu(), ends.float())
  assert torch.equal(codes, ref.codes_of(x.cuda().float(), 127, most[:, None]))
  # one token with each of 127 codes, moved into a block with one of a larger scale
  n = ends.numel() // 2 * 2
  cache = cache8.init_cache(n, 32, 1, 128, "cuda", block=16, weights=True)
  for k in ("key", "value"):
    cache["cached_" + k][:, 0, 0] = torch.arange(128)
    cache[k + "_absmax"][:, 0, 0] = ends[:n].float().cuda()
    cache[k + "_absmax"][:, 0, 1] = ends[:n].float().cuda().roll(n // 3) * 2
  cache["cache_index"].fill_(17)
  cache["token_weight"][:, :, 0] = 1.0
  small, _ = cache8.evict(cache, 2, recent=1)
  old, new = cache["key_absmax"][:, 0, 0], cache["key_absmax"][:, 0, 1]
  want = ref.codes_of(old[:, None], cache["cached_key"][:, 0, 0], torch.maximum(old, new)[:, None])
  want = torch.where((old >= new)[:, None], cache["cached_key"][:, 0, 0], want)
  assert torch.equal(small["cached_key"][:, 0, 0], want) and torch.equal(small["cached_value"][:, 0, 0], want)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(bad, dtype):
  c = dict(b=1, h=1, group=1, dim=64, slots=64, block=16, starts=[20], count=1)
  cache, query, key, value, _ = plain.inputs(c, "cuda", dtype)
  hide = torch.ones(1, 64, dtype=torch.bool, device="cuda")
  hide[0, 16:32] = False  # the block that gets it
  new = [t.cuda().to(dtype) for t in plain.tokens(1, 1, 1, 64)]
  want = cache8.attention(query, {k: v.clone() for k, v in cache.items()}, *new, key_mask=hide)
  for which in (key, value):
    worse = {k: v.clone() for k, v in cache.items()}
    which[0, 0, 0, 3] = bad
    assert torch.equal(cache8.attention(query, worse, key, value, key_mask=hide), want)
    assert cache8.attention(query, worse, key, value).isnan().all()
    which[0, 0, 0, 3] = 1


def test_biases_of_the_lowest_value_and_of_minus_infinity():
  c = dict(b=1, h=2, group=1, dim=64, slots=64, block=16, starts=[12], count=1)
  cache, query, key, value, _ = plain.inputs(c, "cuda", torch.float32)
  low = torch.full((2, 32), torch.finfo(torch.float32).min, device="cuda")
  out = cache8.attention(query * 0, cache, key, value, bias_table=low)
  v = ref.cache8_values(cache, "value", torch.float64)[0, :, :13].mean(1)
  assert torch.allclose(out[0, 0].double(), v, rtol=0, atol=2.0 ** -20 * v.abs().max().item() * 16)
  assert (cache8.attention(query, cache, key, value, bias_table=torch.full_like(low, -math.inf)) == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_pieces_of_wider_tensors(dtype):
  c = dict(b=2, h=2, group=1, dim=64, slots=64, block=16, starts=[9, 30], count=3)
  cache, query, key, value, _ = plain.inputs(c, "cuda", dtype)
  want = cache8.attention(query, {k: v.clone() for k, v in cache.items()}, key, value)
  qkv = torch.cat([t.reshape(2, 3, 128) for t in (query, key, value)] + [torch.zeros(2, 3, 1, device="cuda", dtype=dtype)], 2)
  for parts in (
      [p.unflatten(2, (2, 64)) for p in qkv[..., :384].split(128, 2)],  # rows of an odd length
      [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (query, key, value)],
      [t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0) for t in (query, key, value)],  # channels far apart
      [torch.cat([t.flatten(), t.flatten()[:1]])[1:].roll(1).view_as(t) for t in (query, key, value)]):
    again = {k: v.clone() for k, v in cache.items()}
    assert torch.equal(cache8.attention(*[parts[0], again, *parts[1:]]), want)


def test_mask_types_and_widths():
  c = dict(b=2, h=1, group=1, dim=64, slots=64, block=16, starts=[40, 30], count=2, cross=True)
  cache, query, _, _, _ = plain.inputs(c, "cuda", torch.float32)
  mask = torch.rand(2, 33, device="cuda") > 0.5
  want = cache8.attention(query, cache, key_mask=mask, causal=False)
  wide = torch.zeros(2, 64, device="cuda", dtype=torch.bool)
  wide[:, :33] = mask
  for m in (mask.int() * 256, mask.float(), wide, wide.t().contiguous().t()):
    assert torch.equal(cache8.attention(query, cache, key_mask=m, causal=False), want)
  assert (cache8.attention(query, cache, key_mask=mask[:, :0], causal=False) == 0).all()


@pytest.mark.parametrize("c", plain.EVICT, ids=range(len(plain.EVICT)))
@pytest.mark.parametrize("special", [False, True])
def test_evict(c, special):
  launches(lambda: plain.check_evict(c, "cuda", special))


@pytest.mark.parametrize("slots,keep,recent", [(4096, 700, 33), (8192, 3000, 0), (16384, 129, 128), (20480, 517, 5),
                                               (65536, 1000, 17), (66048, 257, 100)])
@pytest.mark.parametrize("special", [False, True])
def test_evict_from_long_caches(slots, keep, recent, special):
  launches(lambda: plain.check_evict(dict(b=2, h=1, dim=64, slots=slots, block=64, starts=[slots - 7, slots // 2], keep=keep,
                                          recent=recent, to_block=128), "cuda", special))


@pytest.mark.parametrize("slots,keep,recent", [(2048, 256, 256), (2048, 257, 3), (1024, 1000, 1), (640, 256, 0), (2048, 1, 1)])
@pytest.mark.parametrize("dim,to_block", [(64, 16), (128, 128)])
def test_evict_in_one_launch_and_two(slots, keep, recent, dim, to_block):
  for special in (False, True):
    launches(lambda: plain.check_evict(dict(b=3, h=2, dim=dim, slots=slots, block=32, starts=[slots, slots - 333, 200], keep=keep,
                                            recent=recent, to_block=to_block), "cuda", special))


@pytest.mark.parametrize("rows,k,n", [(1, 16, 8), (3, 17, 5), (5, 1, 3), (2, 300, 130), (33, 129, 257), (257, 64, 40),
                                      (130, 513, 300)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear8(rows, k, n, dtype):
  launches(lambda: plain.check_linear(rows, k, n, dtype, rows % 2 == 1, "cuda"))


@pytest.mark.parametrize("rows,k,n", [(1, 1024, 2816), (16, 4096, 130), (17, 2049, 517), (64, 128, 128), (61, 16384 + 8, 96),
                                      (129, 700, 1000), (300, 16400, 40), (2600, 160, 2040), (2304, 96, 2304)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear8_of_every_tile(rows, k, n, dtype):
  """Sizes on both sides of the choices of tiles and pieces, against the statement (exact sums, rounded once)."""
  gen = torch.Generator("cuda").manual_seed(rows)
  randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
  weight = F.quantize_weight(randn(k, n))
  x, r = randn(rows, k).to(dtype), randn(rows, n).to(dtype)
  for residual in (None, r):
    y = launches(lambda: F.linear8(x, weight, residual))  # noqa: B023
    want = ref.linear8(x.double(), weight.codes[:, :k], weight.absmax, None if residual is None else residual.double())
    # eight roundings in 32 bits of the product, and the last one
    size = (want if residual is None else want - residual.double()).abs() + want.abs()
    info = torch.finfo(dtype)
    off = (y.double() - want).abs() - info.eps / 2 * want.abs()
    # (results below the smallest normal number are a whole number of its steps: half a step is smallest * eps / 2)
    assert bool((off <= size * 2.0 ** -21 * (1 + info.eps) + info.smallest_normal * info.eps / 2).all())


@pytest.mark.parametrize("rows,k,n", [(1, 528, 19100), (60, 130, 40000), (128, 257, 19001), (129, 64, 19100), (200, 300, 9400)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear8_of_wide_outputs(rows, k, n, dtype):
  """Few rows into more channels than one round of the SMs takes."""
  gen = torch.Generator("cuda").manual_seed(rows)
  randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
  weight = F.quantize_weight(randn(k, n))
  x, r = randn(rows, k).to(dtype), randn(rows, n).to(dtype)
  for residual in (None, r):
    y = launches(lambda: F.linear8(x, weight, residual))  # noqa: B023
    want = ref.linear8(x.double(), weight.codes[:, :k], weight.absmax, None if residual is None else residual.double())
    # eight roundings in 32 bits of the product, and the last one
    size = (want if residual is None else want - residual.double()).abs() + want.abs()
    info = torch.finfo(dtype)
    off = (y.double() - want).abs() - info.eps / 2 * want.abs()
    # (results below the smallest normal number are a whole number of its steps: half a step is smallest * eps / 2)
    assert bool((off <= size * 2.0 ** -21 * (1 + info.eps) + info.smallest_normal * info.eps / 2).all())


@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 16, 5), (2, 8192, 33), (2, 8208, 33), (2, 4096, 5000), (1, 32768, 70), (1, 32784, 70),
                                      (1, 2047, 9001), (2, 515, 4799), (1, 12000, 17)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear8_of_one_row_and_two(rows, k, n, dtype):
  gen = torch.Generator("cuda").manual_seed(rows)
  randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
  weight = F.quantize_weight(randn(k, n))
  x, r = randn(rows, k).to(dtype), randn(rows, n).to(dtype)
  for residual in (None, r):
    y = launches(lambda: F.linear8(x, weight, residual))  # noqa: B023
    want = ref.linear8(x.double(), weight.codes[:, :k], weight.absmax, None if residual is None else residual.double())
    # eight roundings in 32 bits of the product, and the last one
    size = (want if residual is None else want - residual.double()).abs() + want.abs()
    info = torch.finfo(dtype)
    off = (y.double() - want).abs() - info.eps / 2 * want.abs()
    # (results below the smallest normal number are a whole number of its steps: half a step is smallest * eps / 2)
    assert bool((off <= size * 2.0 ** -21 * (1 + info.eps) + info.smallest_normal * info.eps / 2).all())


def test_linear8_strides():
  weight = F.quantize_weight(torch.randn(48, 40).cuda())
  x, r = torch.randn(9, 7, 48).cuda().bfloat16(), torch.randn(9, 7, 40).cuda().bfloat16()
  want = F.linear8(x, weight, r)
  wide = torch.zeros(9, 7, 99, device="cuda", dtype=torch.bfloat16)
  wide[..., 1:49], wide[..., 50:90] = x, r
  assert torch.equal(F.linear8(wide[..., 1:49], weight, wide[..., 50:90]), want)
  assert torch.equal(F.linear8(x.transpose(0, 1).contiguous().transpose(0, 1), weight, r), want)
  assert torch.equal(F.linear8(x[0, 0], weight, r[0, 0]), want[0, 0])


def test_linear8_rows_that_are_not_finite():
  weight = F.quantize_weight(torch.randn(64, 40).cuda())
  x = torch.randn(5, 64).cuda()
  want = F.linear8(x, weight)
  x[1, 3], x[3, 0] = math.nan, -math.inf
  y = F.linear8(x, weight)
  assert y[1].isnan().all() and y[3].isnan().all() and torch.equal(y[::2], want[::2])


@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear8_of_a_row_that_is_not_finite(rows, bad, dtype):
  weight = F.quantize_weight(torch.randn(300, 40).cuda())
  x = torch.randn(rows, 300).cuda().to(dtype)
  want = F.linear8(x, weight)
  x[0, 299] = bad
  y = F.linear8(x, weight)
  assert want.isfinite().all() and y[0].isnan().all() and torch.equal(y[1:], want[1:])
  assert (F.linear8(torch.zeros_like(x), weight) == 0).all()


def test_another_stream_and_two_captures():
  """Two graphs of the same cache's steps, replayed in turn, and a call on another stream."""
  c = dict(b=2, h=2, group=1, dim=64, slots=640, block=32, starts=[300, 500], count=1, weights=True, bias=True)
  cache, query, key, value, kw = plain.inputs(c, "cuda", torch.bfloat16)
  want = cache8.attention(query, {k: v.clone() for k, v in cache.items()}, key, value, **kw)
  torch.cuda.synchronize()
  graphs, outs, caches = [], [], []
  for _ in range(2):
    mine = {k: v.clone() for k, v in cache.items()}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs.append(cache8.attention(query, mine, key, value, **kw))
    graphs.append(g)
    caches.append(mine)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    beside = cache8.attention(query, {k: v.clone() for k, v in cache.items()}, key, value, **kw)
  for _ in range(3):
    for g in graphs:
      g.replay()
  torch.cuda.synchronize()
  assert torch.equal(beside, want) and all(torch.equal(o, want) for o in outs)
  assert torch.equal(caches[0]["token_weight"], caches[1]["token_weight"])


def test_decode_evict_decode():
  """A run as a server makes it: prompts, tokens one at a time, an eviction, more tokens; beside the statements."""
  b, heads, kv, dim, slots = 3, 6, 2, 64, 160
  table = torch.randn(heads, 32)
  gen = torch.Generator().manual_seed(0)
  both = [cache8.init_cache(b, slots, kv, dim, d, block=16, weights=True, positions=True) for d in ("cuda", "cpu")]
  lengths = torch.tensor([90, 3, 41], dtype=torch.int32)
  prompt = [torch.randn(b, 90, kv, dim, generator=gen).bfloat16() for _ in range(2)]
  for cache in both:
    d = cache["cached_key"].device
    cache8.append_(cache, *[t.to(d) for t in prompt], lengths.to(d))
    cache["cache_index"] += lengths.to(d)
  w = torch.nn.Parameter(torch.randn(heads * dim, heads * dim, generator=gen) / 20)
  weights = [F.quantize_weight(w.cuda()), F.quantize_weight(w)]
  for step in range(60):
    q = (torch.randn(b, 1, heads, dim, generator=gen) / 4).bfloat16()
    k, v = [torch.randn(b, 1, kv, dim, generator=gen).bfloat16() for _ in range(2)]
    outs = []
    for i, cache in enumerate(both):
      d = cache["cached_key"].device
      x = cache8.attention(q.to(d), cache, k.to(d), v.to(d), bias_table=table.to(d))
      cache["cache_index"] += 1
      outs.append((x.cpu(), F.linear8(x.flatten(2), weights[i]).cpu()))
    assert torch.allclose(outs[0][0].float(), outs[1][0].float(), rtol=2.0 ** -7, atol=2.0 ** -8)
    assert torch.equal(both[0]["cached_key"].cpu(), both[1]["cached_key"])
    if step in (20, 45):
      # (weights of 32 bits may differ in the last place: both go by the same ones)
      both[0]["token_weight"].copy_(both[1]["token_weight"])
      both = [cache8.evict(c, 40, recent=8, out=cache8.init_cache(b, 96, kv, dim, c["cached_key"].device, block=16,
                                                                  weights=True, positions=True))[0] for c in both]
      assert all(torch.equal(both[0][n].cpu(), both[1][n]) for n in both[0])


@pytest.mark.parametrize("c", [
    dict(b=2, h=2, group=4, dim=128, slots=8192, block=64, starts=[8000, 4097], count=1, weights=True),
    dict(b=1, h=1, group=1, dim=64, slots=70000 // 16 * 16, block=16, starts=[69000], count=1, bias=True),
    dict(b=2, h=1, group=2, dim=128, slots=4096, block=32, starts=[2048, 3901], count=150, bias=True, weights=True),
], ids=range(3))
@pytest.mark.parametrize("dtype", TYPES)
def test_long(c, dtype):
  cache, query, key, value, kw = plain.inputs(c, "cuda", dtype)
  other = {k: v.clone() for k, v in cache.items()}
  out = launches(lambda: cache8.attention(query, cache, key, value, **kw))
  ref.cache8_append(other, key, value)
  wide = {k: kw[k] for k in ("bias_table", "key_mask", "causal", "scale")}
  want = ref.cache8_attention(query.double(), other, c["count"], **wide)
  assert torch.equal(cache["cached_key"], other["cached_key"]) and torch.equal(cache["value_absmax"], other["value_absmax"])
  # |v| is at most 3, and a query's score below 2^6 by its values
  assert plain.within(out, want.cpu(), torch.full_like(want.cpu(), 3.0), 64.0, c["dim"], c["slots"])
  if c.get("weights"):
    assert torch.allclose(cache["token_weight"], other["token_weight"], rtol=1e-4, atol=1e-7)


def test_offsets_behind_32_bits():
  """A cache whose last row lies behind 2^31 codes."""
  b, slots = 5, 1 << 19
  cache = cache8.init_cache(b, slots, 8, 128, "cuda", block=128, weights=True)
  cache["cache_index"].copy_(torch.tensor([0, 0, 0, 0, slots - 9]))
  key = torch.randn(b, 8, 8, 128, device="cuda", dtype=torch.bfloat16)
  cache8.append_(cache, key, key)
  codes, most = cache["cached_key"][4, :, slots - 9:slots - 1], cache["key_absmax"][4, :, -1]
  assert torch.equal(codes, ref.codes_of(key[4].float().transpose(0, 1), 127, most[:, None, None]))
  cache["cache_index"] += 8
  cache["cache_index"][4] = slots
  hide = torch.zeros(b, slots, dtype=torch.bool, device="cuda")
  hide[:4, :8], hide[4, slots - 9:slots - 1] = True, True
  q = torch.randn(b, 1, 8, 128, device="cuda", dtype=torch.bfloat16) / 8
  out = cache8.attention(q, cache, key_mask=hide, causal=False)
  v = torch.stack([cache["cached_value"][i, :, :8] if i < 4 else cache["cached_value"][4, :, slots - 9:slots - 1]
                   for i in range(b)]).float() * (key.float().abs().amax((1, 3))[:, :, None, None] / 127)
  p = torch.softmax(torch.einsum("blhd,bhsd->bhls", q.float(), v), -1)
  want = torch.einsum("bhls,bhsd->blhd", p, v)
  assert torch.allclose(out.float(), want, rtol=2.0 ** -8, atol=2.0 ** -9 * v.abs().max().item())
  cache["token_weight"][4, :, slots - 1] = 1.0
  small, kept = cache8.evict(cache, 4, recent=0, out=cache8.init_cache(b, 16, 8, 128, "cuda", block=16, weights=True,
                                                                       positions=True))
  assert (kept[4] >= slots - 9).all() and (small["dropped"][4] == slots - 4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [
    dict(b=2, h=1, group=3, dim=64, slots=160, block=32, starts=[120, 0], count=3, mask=True, weights=True),
    dict(b=2, h=2, group=16, dim=128, slots=96, block=16, starts=[61, 15], count=1, bias=True, positions=True),
    dict(b=1, h=2, group=11, dim=64, slots=400, block=16, starts=[366], count=3, bias=True, weights=True),
    dict(b=3, h=1, group=1, dim=128, slots=208, block=16, starts=[200, 0, 77], count=65, weights=True),
    dict(b=2, h=1, group=2, dim=64, slots=192, block=64, starts=[128, 192], count=32, cross=True, mask=True),
    dict(b=1, h=1, group=5, dim=128, slots=144, block=16, starts=[17], count=26, mask=True, bias=True),
    dict(b=2, h=1, group=1, dim=64, slots=272, block=16, starts=[0, 1], count=260, bias=True, weights=True, positions=True),
    dict(b=2, h=1, group=2, dim=128, slots=80, block=16, starts=[64, 3], count=129, own=True),
], ids=range(8))
def test_many_rows(c, dtype):
  """9 to 520 query rows a key head: below and above what a warp, half of a CTA's warps and all of them take."""
  launches(lambda: plain.check_attention(c, "cuda", dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [
    dict(b=4, h=2, group=1, dim=64, slots=2064, block=16, starts=[0, 2063, 5, 1030], count=1, bias=True, weights=True),
    dict(b=3, h=1, group=4, dim=64, slots=2080, block=32, starts=[2000, 0, 700], count=2, weights=True, positions=True, bias=True),
    dict(b=2, h=3, group=3, dim=64, slots=2064, block=16, starts=[1500, 17], count=1, mask=True, weights=True),
    dict(b=3, h=2, group=1, dim=128, slots=2176, block=128, starts=[0, 2176, 901], count=3, cross=True, mask=True),
    dict(b=2, h=1, group=7, dim=128, slots=2112, block=64, starts=[2111, 1], count=1, bias=True, positions=True),
    dict(b=1, h=1, group=2, dim=128, slots=2064, block=16, starts=[3], count=4, own=True, weights=True),
], ids=range(6))
def test_pieces(c, dtype):
  """Caches that are cut into pieces: rows that hold nothing, a token, all; a piece's border inside a row."""
  launches(lambda: plain.check_attention(c, "cuda", dtype))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,count", [(64, 30), (128, 150)])
def test_many_rows_and_values_that_are_not_finite(bad, dtype, dim, count):
  """The last token's block is not finite: the queries before it do not see it, and a mask hides it from all."""
  c = dict(b=1, h=1, group=2, dim=dim, slots=304, block=16, starts=[0], count=count)
  cache, query, key, value, _ = plain.inputs(c, "cuda", dtype)
  cache["cache_index"].fill_(289 - count)  # (the last one begins a block)
  hide = torch.ones(1, 304, dtype=torch.bool, device="cuda")
  hide[0, 288:] = False
  fresh = lambda: {n: t.clone() for n, t in cache.items()}  # noqa: E731
  masked, plainly = cache8.attention(query, fresh(), key, value, key_mask=hide), cache8.attention(query, fresh(), key, value)
  assert masked.isfinite().all() and plainly.isfinite().all()
  for which in (key, value):
    which[0, -1, 0, 3] = bad
    assert torch.equal(cache8.attention(query, fresh(), key, value, key_mask=hide), masked)
    out = cache8.attention(query, fresh(), key, value)
    assert out[:, -1].isnan().all() and torch.equal(out[:, :-1], plainly[:, :-1])
    which[0, -1, 0, 3] = 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,count,slots", [(64, 1, 64), (128, 2, 2112), (64, 40, 64), (128, 200, 256)])
def test_a_hidden_block_of_the_largest_values(dtype, dim, count, slots):
  """Values of 3e38 that a mask hides beside seen ones of 1e-3: their ratio is no number in 32 bits."""
  c = dict(b=1, h=1, group=2, dim=dim, slots=slots, block=16, starts=[64], count=count, own=True)
  cache, query, _, _, _ = plain.inputs(c, "cuda", dtype)
  hide = torch.ones(1, slots, dtype=torch.bool, device="cuda")
  hide[0, 16:32] = False
  cache["value_absmax"].fill_(1e-3)
  want = cache8.attention(query, cache, key_mask=hide, causal=False)
  cache["value_absmax"][0, 0, 1] = cache["key_absmax"][0, 0, 1] = 3e38
  assert want.isfinite().all() and (want != 0).any()
  assert torch.equal(cache8.attention(query, cache, key_mask=hide, causal=False), want)


def test_many_rows_and_biases_of_the_lowest_value():
  c = dict(b=1, h=2, group=1, dim=64, slots=64, block=16, starts=[12], count=20)
  cache, query, key, value, _ = plain.inputs(c, "cuda", torch.float32)
  low = torch.full((2, 32), torch.finfo(torch.float32).min, device="cuda")
  out = cache8.attention(query * 0, cache, key, value, bias_table=low)
  held = ref.cache8_values(cache, "value", torch.float64)[0]
  for i in (0, 7, 19):
    v = held[:, :13 + i].mean(1)
    assert torch.allclose(out[0, i].double(), v, rtol=0, atol=2.0 ** -20 * held.abs().max().item() * 16)
  assert (cache8.attention(query, cache, key, value, bias_table=torch.full_like(low, -math.inf)) == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_of_any_stride(dtype):
  c = dict(b=2, h=2, group=3, dim=64, slots=128, block=16, starts=[9, 30], count=15)
  cache, query, _, _, _ = plain.inputs(dict(c, own=True), "cuda", dtype)
  want = cache8.attention(query, cache)
  wide = torch.cat([query.flatten(2), torch.zeros(2, 15, 1, device="cuda", dtype=dtype)], 2)
  for q in (wide[..., :384].unflatten(2, (6, 64)), query.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3),
            torch.cat([query.flatten(), query.flatten()[:1]])[1:].roll(1).view_as(query)):
    assert torch.equal(cache8.attention(q, cache), want)


def check_some_rows(c, rows, dtype=torch.bfloat16):
  """As check_attention, for some rows of a batch."""
  cache, query, key, value, kw = plain.inputs(c, "cuda", dtype)
  before = cache["token_weight"].clone() if c.get("weights") else None
  out = launches(lambda: cache8.attention(query, cache, key, value, **kw))
  for i in rows:
    held = {n: t[i:i + 1] for n, t in cache.items()}
    mask = None if kw["key_mask"] is None else kw["key_mask"][i:i + 1].cpu()
    want, size, high, weight = plain.attention_oracle(query[i:i + 1], held, [c["starts"][i]], 0 if key is None else c["count"],
                                                      kw["bias_table"], mask=mask, causal=kw["causal"], scale=kw["scale"])
    assert plain.within(out[i:i + 1], want, size, high, c["dim"], c["slots"]), i
    if before is not None:
      new = slice(c["starts"][i], c["starts"][i] + (0 if key is None else c["count"]))
      before[i, :, new] = 0
      each = 2 * ((c["dim"] + 16) * 2.0 ** -24 + 2.0 ** -21) * high + (c["slots"] + 64) * 2.0 ** -24 + 2.0 ** -20
      off = (cache["token_weight"][i].cpu().double() - before[i].cpu().double() - weight[0]).abs()
      assert (off <= each * weight[0] + 2.0 ** -24 * cache["token_weight"][i].cpu().double().abs() + 2.0 ** -120).all(), i


def test_more_rows_than_a_launch_takes():
  starts = [(7 * i) % 1024 for i in range(2050)]
  for count in (1, 9):
    check_some_rows(dict(b=2050, h=1, group=1, dim=64, slots=1040, block=16, starts=starts, count=count), [0, 2047, 2048, 2049])
  # and in pieces
  gen = torch.Generator("cuda").manual_seed(0)
  cache = cache8.init_cache(2050, 8208, 1, 64, "cuda", block=16)
  for n in ("key", "value"):
    cache["cached_" + n].copy_(torch.randint(-127, 128, cache["cached_" + n].shape, generator=gen, device="cuda", dtype=torch.int8))
    cache[n + "_absmax"].fill_(2.0)
  starts = [(31 * i) % 999 for i in range(2050)]
  cache["cache_index"].copy_(torch.tensor(starts))
  query, key, value = [torch.randn(2050, 1, 1, 64, generator=gen, device="cuda").bfloat16() / 4 for _ in range(3)]
  out = launches(lambda: cache8.attention(query, cache, key, value))
  for i in (0, 1, 2046, 2047, 2048, 2049):
    want, size, high, _ = plain.attention_oracle(query[i:i + 1], {n: t[i:i + 1] for n, t in cache.items()}, [starts[i]], 1)
    assert plain.within(out[i:i + 1], want, size, high, 64, 8208), i


def test_more_scores_than_a_launch_takes():
  """The weights of 34 rows come from 1.06 GiB of scores."""
  starts = [(397 * i) % 2048 + 100 for i in range(34)]
  check_some_rows(dict(b=34, h=8, group=8, dim=64, slots=16384, block=128, starts=starts, count=8, weights=True), [0, 31, 32, 33])


def test_tables_beyond_the_kernels():
  """Biases of more heads than shared memory holds, and of longer distances: the statements."""
  for heads, group, far in ((2, 150, 128), (2, 2, 2000)):
    cache = plain.make(1, heads, 48, 64, 16, [40], device="cuda")
    query = torch.randn(1, 1, heads * group, 64, device="cuda") / 8
    table = torch.randn(heads * group, 32, device="cuda")
    out = cache8.attention(query, cache, bias_table=table, max_distance=far)
    want, size, high, _ = plain.attention_oracle(query, cache, [40], 0, table, far=far)
    # (the statements round each score's and each sum's products in another order: as many roundings at most)
    assert plain.within(out, want, size, high, 64, 48)


def test_evict_and_products_captured_beside_each_other():
  """Each captured once and replayed on its own stream, while the same calls run on the current one."""
  cache = plain.make(2, 2, 512, 64, 32, [500, 77], weights=True, positions=True, device="cuda")
  room = lambda: cache8.init_cache(2, 256, 2, 64, "cuda", block=32, weights=True, positions=True)  # noqa: E731
  weight = F.quantize_weight(torch.randn(320, 640).cuda())
  xs = [torch.randn(n, 320).cuda().bfloat16() for n in (1, 40, 700)]
  small, kept = cache8.evict(cache, 200, recent=20, out=room())
  want = [F.linear8(x, weight) for x in xs]
  torch.cuda.synchronize()
  streams, graphs, got = [torch.cuda.Stream() for _ in range(2)], [], []
  for _ in range(2):
    into, g = room(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      got.append((*cache8.evict(cache, 200, recent=20, out=into), [F.linear8(x, weight) for x in xs]))
    graphs.append(g)
  for _ in range(3):
    for s, g in zip(streams, graphs):
      with torch.cuda.stream(s):
        g.replay()
    again, again_kept = cache8.evict(cache, 200, recent=20, out=room())
    here = [F.linear8(x, weight) for x in xs]
  torch.cuda.synchronize()
  for into, slots, ys in got + [(again, again_kept, here)]:
    assert torch.equal(slots, kept) and all(torch.equal(into[n], small[n]) for n in small)
    assert all(torch.equal(y, w) for y, w in zip(ys, want))


def test_threads():
  """Calls of several threads at once, each with a stream and a cache of its own."""
  c = dict(b=3, h=2, group=2, dim=64, slots=1600, block=32, starts=[1500, 3, 700], count=1, weights=True, bias=True)
  cache, query, key, value, kw = plain.inputs(c, "cuda", torch.bfloat16)
  chunk = torch.randn(3, 30, 4, 64, device="cuda", dtype=torch.bfloat16) / 8
  weight, x = F.quantize_weight(torch.randn(64, 80).cuda()), torch.randn(9, 64).cuda()

  def run():
    mine = {n: t.clone() for n, t in cache.items()}
    outs = [cache8.attention(query, mine, key, value, **kw), cache8.attention(chunk, mine, causal=False), F.linear8(x, weight)]
    return outs + [mine["token_weight"], cache8.evict(mine, 90, recent=3)[1]]

  want = run()
  torch.cuda.synchronize()
  got = {}

  def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
      for _ in range(20):
        got[i] = run()
      torch.cuda.current_stream().synchronize()

  threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  assert len(got) == 4 and all(torch.equal(a, b) for one in got.values() for a, b in zip(one, want))


@pytest.mark.parametrize("heads,group,count,slots,own", [(5, 8, 300, 32768, False), (2, 8, 1100, 32768, False), (1, 3, 20000, 8208, True)])
def test_one_row_of_more_scores_than_a_launch_takes(heads, group, count, slots, own):
  """Heads, or queries of a head, go in several launches: with the results and weights of one, and a gigabyte of workspace."""
  dim, held = 64, slots - count - 5
  cache = plain.make(1, heads, slots, dim, 16, [held + count if own else held], weights=True, positions=True, device="cuda")
  gen = torch.Generator("cuda").manual_seed(0)
  randn = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()  # noqa: E731
  query, table = randn(1, count, heads * group, dim) / 4, torch.randn(heads * group, 32, generator=gen, device="cuda")
  key, value = (None, None) if own else (randn(1, count, heads, dim), randn(1, count, heads, dim))
  shown = torch.rand(1, slots, generator=gen, device="cuda") > 0.2
  before = cache["token_weight"].double()
  torch.cuda.synchronize()
  start = torch.cuda.memory_allocated()
  torch.cuda.reset_peak_memory_stats()
  out = launches(lambda: cache8.attention(query, cache, key, value, bias_table=table, key_mask=shown))
  assert torch.cuda.max_memory_allocated() - start < 1.25 * 2 ** 30
  before[:, :, held:held + count] *= own
  added = torch.zeros_like(before)
  values = {n: ref.cache8_values(cache, n, torch.float64) for n in ("key", "value")}
  slot = torch.arange(slots, device="cuda")
  for i in range(0, count, 500):  # in 64 bits
    for h in range(heads):
      q = query[0, i:i + 500, h * group:(h + 1) * group].double()
      s = torch.einsum("lgd,sd->gls", q, values["key"][0, h])
      own_at = held + i + torch.arange(q.shape[0], device="cuda")
      back = cache["token_position"][0, h].long() - (own_at + cache["dropped"].long())[:, None]
      s += table[h * group:(h + 1) * group].double()[:, ref.relative_position_bucket(back, False, 32, 128)]
      s.masked_fill_((slot > own_at[:, None]) | ~shown, -math.inf)
      p = torch.softmax(s, 2).nan_to_num()  # (queries in front of all that is held see nothing)
      added[0, h] += p.sum((0, 1))
      want = torch.einsum("gls,sd->lgd", p, values["value"][0, h])
      # |v| is at most 3; a score's products are below 2^6
      size = torch.full_like(want, 3.0)
      assert plain.within(out[0, i:i + 500, h * group:(h + 1) * group], want.cpu(), size.cpu(), 64.0, dim, slots)
  assert torch.allclose(cache["token_weight"].double(), before + added, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("rows", [148, 149, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_evict_of_as_many_heads_as_the_sms_take_at_a_time_and_more(rows, dim):
  """Four heads a row: 592 CTAs, and more."""
  starts = [(37 * i) % 96 for i in range(rows)]
  launches(lambda: plain.check_evict(dict(b=rows, h=4, dim=dim, slots=96, block=16, starts=starts, keep=30, recent=7, to_block=16),
                                     "cuda", False))


def test_weights_of_more_slots_than_65535_blocks():
  """16.8 million slots, of which a mask shows a few: the first, one in the middle, those at the end."""
  slots = 65536 * 256 + 64
  cache = cache8.init_cache(1, slots, 1, 64, "cuda", block=64, weights=True)
  at = torch.tensor([0, 12345678, 65535 * 256 + 7, slots - 1], device="cuda")
  cache["cached_value"][0, 0, at] = torch.randint(-127, 128, (4, 64), device="cuda", dtype=torch.int8)
  cache["value_absmax"][0, 0, at // 64] = 1.0
  cache["cache_index"].fill_(slots)
  shown = torch.zeros(1, slots, dtype=torch.bool, device="cuda")
  shown[0, at] = True
  out = launches(lambda: cache8.attention(torch.randn(1, 1, 1, 64, device="cuda"), cache, key_mask=shown))
  # (keys of 0: each has a quarter)
  want = cache["cached_value"][0, 0, at].double().mean(0) / 127
  assert torch.allclose(out[0, 0, 0].double(), want, rtol=0, atol=2.0 ** -21)
  assert torch.allclose(cache["token_weight"][0, 0, at], torch.full((4,), 0.25, device="cuda"), rtol=2.0 ** -21)
  assert cache["token_weight"].sum(dtype=torch.float64).item() == pytest.approx(1.0, rel=2.0 ** -20)
