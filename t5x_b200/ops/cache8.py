"""A key/value cache held in 8 bits: appending tokens, attention, eviction by attention weight.

The cache is a dict of tensors like the other decode caches of the models (rows first, so that beams are expanded and
gathered as ever), in blocks of 16, 32, 64 or 128 tokens of a head that share a scale:

* `cached_key`, `cached_value`: int8 [rows, heads, slots, head_dim];
* `key_absmax`, `value_absmax`: fp32 [rows, heads, slots / block], the largest absolute value of a block. A code c
  stands for c * absmax / 127. A value that is not finite makes its block NaN. (Attention adds up to 2^32 times a
  value before it divides: seen values beyond 2^96 may come out infinite.);
* `cache_index`: int32, tokens that a row holds ([rows], or one for all). Slots from there on are not read;
* `token_weight`, optional: fp32 [rows, heads, slots], the attention that each token got so far;
* `token_position` int32 [rows, heads, slots] and `dropped` int32 [rows], optional: positions of the tokens, and tokens
  evicted, where slots are not positions (any more).

As in the other caches, `append_` and `attention` write at `cache_index`, and the caller moves it on. Tokens beyond the
last slot are left out. On CUDA, over bf16, fp16 or fp32 queries and head dims of 64 and 128, the kernels of
csrc/cache8.cu and csrc/cache8_attention.cu run; anything else runs the PyTorch statements in
:mod:`t5x_b200.ops.reference`. There is no backward pass.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from t5x_b200.ops import functional as F
from t5x_b200.ops import native
from t5x_b200.ops import reference as ref

BLOCKS = (16, 32, 64, 128)
_TENSORS = {"cached_key": torch.int8, "cached_value": torch.int8, "key_absmax": torch.float32,
            "value_absmax": torch.float32, "cache_index": torch.int32, "token_weight": torch.float32,
            "token_position": torch.int32, "dropped": torch.int32}


def init_cache(batch: int, max_len: int, heads: int, head_dim: int, device=None, *, block: int = 32,
               weights: bool = False, positions: bool = False) -> dict:
  """An empty cache for `max_len` tokens (filled up to whole blocks) of `heads` key heads. `weights`: attention weight is
  added up by token; `positions`: tokens carry their positions."""
  if block not in BLOCKS:
    raise ValueError(f"blocks of {block} tokens: one of {BLOCKS}")
  if min(batch, max_len, heads, head_dim) < 1:
    raise ValueError(f"a cache of {batch} rows, {max_len} tokens, {heads} heads of {head_dim}")
  blocks = -(-max_len // block)
  by_slot = (batch, heads, blocks * block)
  zeros = lambda shape, name: torch.zeros(shape, dtype=_TENSORS[name], device=device)  # noqa: E731
  cache = {n: zeros((*by_slot, head_dim), n) for n in ("cached_key", "cached_value")}
  cache |= {n: zeros((batch, heads, blocks), n) for n in ("key_absmax", "value_absmax")}
  cache["cache_index"] = zeros((batch,), "cache_index")
  if weights:
    cache["token_weight"] = zeros(by_slot, "token_weight")
  if positions:
    cache["token_position"], cache["dropped"] = zeros(by_slot, "token_position"), zeros((batch,), "dropped")
  return cache


def _check_cache(cache, what: str) -> None:
  """Raises unless the tensors of a cache fit each other."""
  try:
    codes, most = cache["cached_key"], cache["key_absmax"]
    b, h, slots, dim = codes.shape
    blocks = most.shape[2]
    shapes = {"cached_key": codes.shape, "cached_value": codes.shape, "key_absmax": (b, h, blocks),
              "value_absmax": (b, h, blocks), "token_weight": (b, h, slots), "token_position": (b, h, slots), "dropped": (b,)}
    for name, dtype in _TENSORS.items():
      if name not in cache and name in ("token_weight", "token_position", "dropped"):
        continue
      t = cache[name]
      fits = t.shape in ((), (1,), (b,)) if name == "cache_index" else t.shape == shapes[name]
      if not fits or t.dtype != dtype or t.device != codes.device or not t.is_contiguous():
        raise ValueError(f"{what}: `{name}` of a cache of {b} rows, {h} heads, {slots} slots is {dtype} on {codes.device}, "
                         f"contiguous; got {tuple(t.shape)} {t.dtype} on {t.device}")
  except (KeyError, IndexError, AttributeError, TypeError) as e:
    raise ValueError(f"{what}: not a cache in 8 bits ({type(e).__name__}: {e})") from None
  if slots % max(1, blocks) or slots // max(1, blocks) not in BLOCKS:
    raise ValueError(f"{what}: {slots} slots in {blocks} blocks; a block has one of {BLOCKS}")
  if "token_position" in cache and "dropped" not in cache:
    raise ValueError(f"{what}: positions without `dropped`")


def _no_graph(what: str, *tensors) -> None:
  if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
    raise ValueError(f"{what} has no backward pass: detach its inputs or call it under torch.no_grad()")


def _check_tokens(cache, key, value, what: str) -> None:
  b, h, _, dim = cache["cached_key"].shape
  if key.dim() != 4 or key.shape != value.shape or key.dtype != value.dtype or not key.dtype.is_floating_point or \
      (key.shape[0], key.shape[2], key.shape[3]) != (b, h, dim) or key.shape[1] < 1:
    raise ValueError(f"{what}: keys and values are [{b}, tokens, {h}, {dim}] of one type; got {tuple(key.shape)} {key.dtype} "
                     f"and {tuple(value.shape)} {value.dtype}")
  if key.device != cache["cached_key"].device or value.device != key.device:
    raise ValueError(f"{what}: new tokens on {key.device}, the cache on {cache['cached_key'].device}")
  _no_graph(what, key, value)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
  """Whether two contiguous tensors share memory."""
  at, to = a.data_ptr(), b.data_ptr()
  return at < to + b.numel() * b.element_size() and to < at + a.numel() * a.element_size()


def _native_ok(cache, dtype) -> bool:
  """Whether the kernels take the call. (A function transform or a trace sees into the statements, not into kernels.)"""
  codes = cache["cached_key"]
  return codes.is_cuda and codes.shape[3] in (64, 128) and dtype in native.CACHE8_TYPES and codes.numel() > 0 and \
      codes.shape[0] < 65536 and codes.shape[1] < 65536 and codes.shape[0] * codes.shape[1] <= 1 << 24 and \
      not F._transformed()


def append_(cache: dict, key: torch.Tensor, value: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> None:
  """Writes tokens key, value [rows, L, heads, head_dim] behind those that the rows hold, `lengths` [rows] of them where it
  is given (a padded batch of prompts). A block that gets tokens takes the largest absolute value of what it holds and
  gets, and the codes that it held are rounded again, relative to that. Their weight is 0, their position the slot's number
  plus the tokens dropped."""
  _check_cache(cache, "append_")
  _check_tokens(cache, key, value, "append_")
  if lengths is not None and (lengths.shape != key.shape[:1] or lengths.device != key.device or lengths.is_floating_point()):
    raise ValueError(f"append_: lengths are whole numbers [{key.shape[0]}] on {key.device}")
  if not _native_ok(cache, key.dtype):
    return ref.cache8_append(cache, key, value, lengths)
  native.cache8_append(cache, key, value, lengths)


def attention(query: torch.Tensor, cache: dict, key: Optional[torch.Tensor] = None, value: Optional[torch.Tensor] = None, *,
              bias_table: Optional[torch.Tensor] = None, num_buckets: int = 32, max_distance: int = 128,
              key_mask: Optional[torch.Tensor] = None, causal: bool = True, scale: float = 1.0) -> torch.Tensor:
  """softmax(scale q k + bias) v over the tokens of a cache; query [rows, L, query heads, head_dim], as many or a multiple of
  the cache's heads (heads that share keys lie side by side). Returns the query's shape and type.

  key, value [rows, L, heads, head_dim]: the queries' own tokens, appended first (see `append_`; `cache_index` is left to
  the caller). With `causal` the queries are the last L tokens, each of which sees itself and what is before it; without
  it they see everything that is held (a cross attention; beams of an example as further queries).
  bias_table [query heads, num_buckets]: learned biases of the T5 buckets of the distance to a token.
  key_mask [rows, n], n <= slots: slots that are seen; those from n on are hidden. A query that sees nothing has zeros and
  gives no weight. With `token_weight` in the cache the softmax of all queries and heads that share keys is added to it."""
  host = native.host() if query.is_cuda and not F._transformed() else None
  if host is not None and (bias_table is None or (bias_table.dim() == 2 and 2 <= bias_table.shape[1] == num_buckets <= 256 and
                                                  num_buckets // 2 < max_distance < native.CACHE8_DISTANCES)):
    # (the plain call, checked there; anything else comes back as None)
    buckets = None if bias_table is None else native.buckets_of(num_buckets, max_distance)
    out = host.cache8_attention(query, cache, key, value, bias_table, buckets, key_mask, bool(causal), float(scale))
    if out is not None:
      return out
  _check_cache(cache, "attention")
  b, h, slots, dim = cache["cached_key"].shape
  if (key is None) != (value is None):
    raise ValueError("attention: keys and values come together")
  if query.dim() != 4 or query.shape[0] != b or query.shape[3] != dim or query.shape[2] % h or query.shape[2] == 0 or \
      query.shape[1] < 1 or not query.dtype.is_floating_point or query.device != cache["cached_key"].device:
    raise ValueError(f"attention: queries are [{b}, L, a multiple of {h}, {dim}] on {cache['cached_key'].device}; got "
                     f"{tuple(query.shape)} {query.dtype} on {query.device}")
  _no_graph("attention", query, bias_table)
  if key is not None:
    _check_tokens(cache, key, value, "attention")
    if key.shape[1] != query.shape[1] or key.dtype != query.dtype:
      raise ValueError(f"attention: {query.shape[1]} queries {query.dtype}, {key.shape[1]} new tokens {key.dtype}")
  if bias_table is not None:
    if bias_table.dim() != 2 or bias_table.shape[0] < query.shape[2] or bias_table.shape[1] < num_buckets or \
        bias_table.device != query.device:
      raise ValueError(f"bias table {tuple(bias_table.shape)} on {bias_table.device}: {query.shape[2]} heads and "
                       f"{num_buckets} buckets are indexed")
    if not 2 <= num_buckets <= 256 or max_distance <= num_buckets // 2:
      raise ValueError(f"{num_buckets} buckets (2 to 256) for distances up to {max_distance} (over half of the buckets)")
  if key_mask is not None and (key_mask.dim() != 2 or key_mask.shape[0] != b or key_mask.shape[1] > slots or
                               key_mask.device != query.device):
    raise ValueError(f"attention: a mask is [{b}, at most {slots}]; got {tuple(key_mask.shape)}")
  if query.shape[1] * (query.shape[2] // h) > 65535:
    raise ValueError("attention: over 65535 query rows a head")
  if "token_weight" in cache and query.shape[1] * (query.shape[2] // h) * slots >= 1 << 31:
    raise ValueError(f"attention: {query.shape[1]} queries over {slots} slots whose weight is added up; give fewer at a time")
  if not (_native_ok(cache, query.dtype) and (bias_table is None or (
      max_distance < native.CACHE8_DISTANCES and query.shape[2] * num_buckets <= native.CACHE8_BIASES))):
    if key is not None:
      ref.cache8_append(cache, key, value)
    return ref.cache8_attention(query, cache, 0 if key is None else key.shape[1], bias_table, num_buckets, max_distance,
                                key_mask, causal, scale)
  return native.cache8_attention(query, cache, key, value, bias_table, num_buckets, max_distance, key_mask, causal, scale)


def evict(cache: dict, keep: int, *, recent: int = 0, out: Optional[dict] = None) -> Tuple[dict, torch.Tensor]:
  """Keeps `keep` tokens of every head of every row: the last `recent` ones, and of the others those that got most attention
  (`token_weight`; ties go to the lower slot, NaN counts as most), in order. Rows that hold no more keep all.

  Returns (a cache with the kept tokens, their slots int32 [rows, heads, keep] with -1 behind the last). The cache is
  `out`, another cache with weights and positions for at least `keep` tokens, whose slots behind them stay as they were, or
  a new one as large as this. Its blocks take the largest scale that a token brings, and codes from smaller ones are
  rounded again."""
  if out is not None and not F._transformed() and getattr(cache.get("cached_key"), "is_cuda", False):
    host = native.host()
    kept = None if host is None else host.cache8_evict(cache, out, keep, recent)
    if kept is not None:
      return out, kept
  _check_cache(cache, "evict")
  if "token_weight" not in cache:
    raise ValueError("evict: the cache adds up no attention weight (init_cache(..., weights=True))")
  b, h, slots, dim = cache["cached_key"].shape
  if not 1 <= keep or not 0 <= recent <= keep:
    raise ValueError(f"evict: {keep} tokens to keep, the last {recent} among them")
  if out is None:
    block = slots // cache["key_absmax"].shape[2]
    out = init_cache(b, slots, h, dim, cache["cached_key"].device, block=block, weights=True, positions=True)
  else:
    _check_cache(out, "evict")
    to = out["cached_key"]
    if "token_weight" not in out or "token_position" not in out or out["cache_index"].shape != (b,) or \
        (to.shape[0], to.shape[1], to.shape[3], to.device) != (b, h, dim, cache["cached_key"].device):
      raise ValueError(f"evict: `out` is another cache of {b} rows, {h} heads of {dim}, with weights and positions")
    if any(_overlap(out[n], cache[m]) for n in out if n in _TENSORS for m in cache if m in _TENSORS):
      raise ValueError("evict: `out` shares memory with the cache")
  if keep > out["cached_key"].shape[2]:
    raise ValueError(f"evict: {keep} tokens into {out['cached_key'].shape[2]} slots")
  if _native_ok(cache, torch.float32):
    return out, native.cache8_evict(cache, out, keep, recent)
  return out, ref.cache8_evict(cache, out, keep, recent)
