"""What is measured of decoding in 8 bits.

* op "attend": attention over a cache held in 8 bits with a scale for each block of tokens and head, the new
  tokens' keys and values appended in the same call: `cache8.attention`;
* op "evict": the tokens that got most attention, and the last ones, moved into a smaller part of a cache:
  `cache8.evict`;
* op "linear8": a projection in 8-bit integers, activations scaled by token and weights by channel:
  `functional.linear8`.

With `own` false every operator is computed from elementary tensor operations. A cache's codes come out beside the
largest value of their blocks: a code c of a block whose largest is a stands for c * a / 127.
"""
import math

import torch

own = False

BUCKETS, FAR = 32, 128  # relative position buckets, and the distance from which on all share the last


def _attend(batch, heads, kv_heads, dim, room, held, new, block=32, dtype="bfloat16", bias=False, mask=False, moved=False):
  """`new` queries; their tokens are appended unless `held` is "all" (a cross attention). `moved`: the cache has been
  evicted from, its tokens carry positions, and their attention weight is added up."""
  return {"op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "room": room, "held": held,
          "new": new, "block": block, "dtype": dtype, "bias": bias, "mask": mask, "moved": moved}


def _evict(batch, kv_heads, dim, room, keep, recent, block=32):
  return {"op": "evict", "batch": batch, "kv_heads": kv_heads, "dim": dim, "room": room, "keep": keep, "recent": recent,
          "block": block}


def _linear(rows, k, n, dtype="bfloat16", residual=False):
  return {"op": "linear8", "rows": rows, "in": k, "out": n, "dtype": dtype, "residual": residual}


def listed():
  cases = [
      # one sentence, one token of the base size
      ("attend_base_one", _attend(1, 12, 12, 64, 640, "most", 1, bias=True)),
      # a batch of XL size, rows of all lengths, from a cache that has been evicted from
      ("attend_xl_batch", _attend(64, 32, 32, 64, 1024, "ragged", 1, bias=True, moved=True)),
      # long contexts, heads that share keys
      ("attend_long", _attend(8, 64, 8, 128, 65536, "ragged", 1)),
      # a chunk of a prompt behind what is held
      ("attend_chunk", _attend(2, 16, 4, 128, 8192, "most", 125, block=64, dtype="float16")),
      # four beams' cross attention over padded inputs, a model in 32 bits
      ("attend_cross", _attend(16, 16, 16, 64, 512, "all", 4, dtype="float32", mask=True)),
      # one sentence
      ("evict_base_one", _evict(1, 12, 64, 640, 121, 32)),
      # prompts of a batch
      ("evict_batch", _evict(16, 32, 64, 2048, 512, 64)),
      # long contexts
      ("evict_long", _evict(8, 8, 128, 65536, 4096, 512, block=64)),
      # one token, large size
      ("linear8_one", _linear(1, 1024, 2816)),
      # a decode step of a batch, XXL size
      ("linear8_batch", _linear(61, 4096, 10240)),
      # a model in 32 bits, odd sizes
      ("linear8_odd", _linear(509, 2049, 517, dtype="float32", residual=True)),
      # prompts, XXL size
      ("linear8_prompt", _linear(8192, 10240, 4096, residual=True)),
  ]
  return [dict(name=n, **c) for n, c in cases]


def _log_int(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  most = max(work(c)["bytes"] for c in listed())
  while True:
    op = rng.choice(["attend", "evict", "linear8"])
    if op == "attend":
      kv, dim = _log_int(rng, 1, 32), rng.choice([64, 128])
      block = rng.choice([16, 32, 64, 128])
      room = block * _log_int(rng, 1, 65536 // block)
      new = rng.choice([1, 1, 1, _log_int(rng, 1, 256)])
      held = rng.choice(["most", "ragged", "ragged", "all"])
      moved = held != "all" and rng.random() < 0.4
      case = _attend(_log_int(rng, 1, 64), kv * rng.choice([1, 1, 2, 4, 7, 8]), kv, dim, room, held, min(new, room), block,
                     rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), held != "all" and rng.random() < 0.5,
                     held == "all" or rng.random() < 0.2, moved)
      fits = work(case)["flops"] <= 2e12 and case["heads"] * new * room * case["batch"] <= 1.5e9
    elif op == "evict":
      block = rng.choice([16, 32, 64, 128])
      room = block * _log_int(rng, 2, 65536 // block)
      keep = _log_int(rng, 1, room - 1)
      case = _evict(_log_int(rng, 1, 64), _log_int(rng, 1, 32), rng.choice([64, 128]), room, keep, rng.randint(0, keep), block)
      fits = 2 * case["batch"] * case["kv_heads"] * room * case["dim"] <= 4e9
    else:
      case = _linear(_log_int(rng, 1, 8192), _log_int(rng, 16, 10240), _log_int(rng, 16, 32128),
                     rng.choice(["bfloat16", "float32"]), rng.random() < 0.5)
      fits = work(case)["flops"] <= 2 * 8192 * 10240 * 4096
    if fits and work(case)["bytes"] <= most:
      return case


# ----------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------
def _held(case):
  """Tokens that each row of the cache holds before the call: the same for every seed, so that the work is too."""
  b, room, new = case["batch"], case["room"], case.get("new", 0)
  if case["op"] == "evict":
    return [room - (7 * i * i) % (room // 4 + 1) for i in range(b)]
  if case["held"] == "all":
    return [room] * b
  if case["held"] == "most":
    return [min(room - new, room * 4 // 5 + i) for i in range(b)]
  return [int((room - new) * ((i * 0.6180339887) % 1.0)) for i in range(b)]


def _codes(shape, gen):
  return torch.randn(shape, generator=gen, device="cuda").mul_(36).round_().clamp_(-127, 127).to(torch.int8)


def _cache(case, gen, empty=False):
  b, h, room, dim, blocks = case["batch"], case["kv_heads"], case["room"], case["dim"], case["room"] // case["block"]
  cache = {}
  for name in ("key", "value"):
    if empty:
      cache["cached_" + name] = torch.zeros(b, h, room, dim, dtype=torch.int8, device="cuda")
      cache[name + "_absmax"] = torch.zeros(b, h, blocks, device="cuda")
    else:
      cache["cached_" + name] = _codes((b, h, room, dim), gen)
      most = 2.5 + 2 * torch.rand(b, h, blocks, generator=gen, device="cuda")
      cache[name + "_absmax"] = most.bfloat16().float()  # (the largest of values of 16 bits)
  cache["cache_index"] = torch.zeros(b, dtype=torch.int32, device="cuda") if empty else \
      torch.tensor(_held(case), dtype=torch.int32, device="cuda")
  return cache


def _weights(shape, gen):
  """Attention weight that tokens got: a few have most of it, many none at all."""
  w = torch.rand(shape, generator=gen, device="cuda")
  return torch.where(w < 0.3, torch.zeros_like(w), (w - 0.3) ** 6 * 8)


def _positions(case, gen):
  """(positions of the slots, tokens dropped by row): slots in order, some tokens between them gone."""
  b, h, room = case["batch"], case["kv_heads"], case["room"]
  held = torch.tensor(_held(case), device="cuda")
  dropped = torch.randint(0, room + 1, (b,), generator=gen, device="cuda")
  jump = torch.rand(b, h, room, generator=gen, device="cuda") * 2 * dropped[:, None, None] / held.clamp(min=1)[:, None, None]
  most = held[:, None, None] + dropped[:, None, None] - 1 - torch.arange(room - 1, -1, -1, device="cuda")
  at = torch.minimum(torch.arange(room, device="cuda") + jump.cumsum(2).long(), most + (room - held)[:, None, None])
  return at.clamp(min=0).int(), dropped.int()


def prepare(case, seed):
  gen = torch.Generator("cuda").manual_seed(seed)
  randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
  if case["op"] == "evict":
    cache = _cache(case, gen)
    cache["token_weight"] = _weights((case["batch"], case["kv_heads"], case["room"]), gen)
    cache["token_position"], cache["dropped"] = _positions(case | {"held": "most"}, gen)
    out = _cache(case | {"room": -(-case["keep"] // case["block"]) * case["block"] + case["block"]}, gen, empty=True)
    out["token_weight"] = torch.zeros_like(out["cached_key"][..., 0], dtype=torch.float32)
    out["token_position"] = torch.zeros_like(out["cached_key"][..., 0], dtype=torch.int32)
    out["dropped"] = torch.zeros_like(cache["dropped"])
    return {"case": case, "cache": cache, "into": out}
  if case["op"] == "linear8":
    rows, k, n, dtype = case["rows"], case["in"], case["out"], getattr(torch, case["dtype"])
    codes = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device="cuda")  # (a channel's weights fill whole 16 bytes)
    codes[:, :k] = _codes((n, k), gen)
    x = randn(rows, k)
    x[:, ::97] *= 6  # channels that stand out
    return {"case": case, "x": x.to(dtype), "codes": codes, "absmax": (0.08 + 0.05 * torch.rand(n, generator=gen, device="cuda")),
            "residual": randn(rows, n).to(dtype) if case["residual"] else None}
  b, h, kv, dim, new, dtype = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "new", "dtype"))
  dtype = getattr(torch, dtype)
  state = {"case": case, "cache": _cache(case, gen), "query": (randn(b, new, h, dim) * 2 / math.sqrt(dim)).to(dtype)}
  if case["held"] != "all":
    state["key"], state["value"] = randn(b, new, kv, dim).to(dtype), randn(b, new, kv, dim).to(dtype)
  if case["bias"]:
    state["bias"] = randn(h, BUCKETS)
  if case["mask"]:  # inputs of several lengths behind padding; the last row's are all padding where there are several
    seen = torch.arange(case["room"], device="cuda")[None] < \
        (case["room"] * (0.4 + 0.6 * torch.rand(b, 1, generator=gen, device="cuda"))).ceil()
    if b > 2 and case["held"] == "all":
      seen[-1] = False
    state["mask"] = seen
  if case["moved"]:
    state["cache"]["token_weight"] = _weights((b, kv, case["room"]), gen)
    state["cache"]["token_position"], state["cache"]["dropped"] = _positions(case, gen)
  return state


def run(state):
  op = state["case"]["op"]
  if own:
    return _run_own(state)
  if op == "attend":
    return _attend_plain(state)
  return _evict_plain(state) if op == "evict" else _linear_plain(state)


def _run_own(state):
  from t5x_b200.ops import cache8, functional
  case = state["case"]
  if case["op"] == "attend":
    out = cache8.attention(state["query"], state["cache"], state.get("key"), state.get("value"), bias_table=state.get("bias"),
                           num_buckets=BUCKETS, max_distance=FAR, key_mask=state.get("mask"), causal=case["held"] != "all")
    return {"out": out, **_held_values(state["cache"], case["held"] != "all")}
  if case["op"] == "evict":
    into, kept = cache8.evict(state["cache"], case["keep"], recent=case["recent"], out=state["into"])
    return {"kept": kept, **into}
  weight = functional.Weight8(state["codes"], state["absmax"], case["in"])
  return functional.linear8(state["x"], weight, residual=state["residual"])


def _held_values(cache, changed):
  """The parts of a cache that an attention with new tokens changes."""
  return {k: v for k, v in cache.items() if k not in ("cache_index", "dropped")} if changed else {}


# ----------------------------------------------------------------------------
# Plain forms
# ----------------------------------------------------------------------------
def _round(real, whole, most):
  """real * whole / most to the nearest whole number (in 64 bits: in 32 a value next to a border may get to its other side)."""
  return torch.nan_to_num(torch.round(real.double() * whole / most), nan=0.0).clamp(-127, 127)


def _append_plain(case, cache, name, new):
  """Blocks that get tokens: the largest of what they hold and get, all codes relative to it."""
  codes, most = cache["cached_" + name], cache[name + "_absmax"]
  b, h, room, dim = codes.shape
  block, count, at = case["block"], new.shape[1], cache["cache_index"].long()
  first = at // block
  touched = (count + block - 2) // block + 1
  blocks = first[:, None] + torch.arange(touched, device="cuda")  # [B, blocks]
  slots = (blocks[:, :, None] * block + torch.arange(block, device="cuda")).view(b, -1)  # [B, S]
  place = slots - at[:, None]  # of the new token, where there is one
  is_new = (place >= 0) & (place < count) & (slots < room)
  is_old = (place < 0) & (slots < room)
  gets = is_new.view(b, touched, block).any(2)
  keeps = is_old.view(b, touched, block).any(2)
  x = new.float().transpose(1, 2).gather(2, place.clamp(0, count - 1)[:, None, :, None].expand(b, h, -1, dim))
  x = torch.where(is_new[:, None, :, None], x, torch.zeros_like(x))
  inside = blocks.clamp(max=room // block - 1)[:, None].expand(b, h, touched)
  before = torch.where(keeps[:, None], most.gather(2, inside), torch.zeros_like(most[:, :, :1]))
  after = torch.maximum(before, x.abs().view(b, h, touched, -1).amax(3))
  each = lambda a: a.repeat_interleave(block, 2)[..., None]  # noqa: E731
  where = slots.clamp(max=room - 1)[:, None, :, None].expand(b, h, -1, dim)
  old = codes.gather(2, where).float()
  again = torch.where(each(before == after), old, _round(each(before), old, each(after)))
  fresh = _round(x, 127, each(after))
  both = torch.where(is_new[:, None, :, None], fresh, torch.where((is_old & gets.repeat_interleave(block, 1))[:, None, :, None],
                                                                  again, old)).to(torch.int8)
  rows = torch.arange(b, device="cuda")[:, None]
  row, s = (rows + 0 * slots)[slots < room], slots[slots < room]
  codes[row, :, s] = both.transpose(1, 2)[slots < room]
  row, k = (rows + 0 * blocks)[gets], blocks[gets]
  most[row, :, k] = after.transpose(1, 2)[gets]


def _bucket(distance):
  """The bucket of a key so many positions back."""
  d = distance.clamp(min=0)
  exact = BUCKETS // 2
  far = exact + (torch.log(d.double().clamp(min=1) / exact) / math.log(FAR / exact) * (BUCKETS - exact)).long()
  return torch.where(d < exact, d, far.clamp(max=BUCKETS - 1))


def _attend_plain(state):
  case, cache, q = state["case"], state["cache"], state["query"]
  b, new, h, dim = q.shape
  kv, room, index = case["kv_heads"], case["room"], cache["cache_index"].long()
  slot = torch.arange(room, device="cuda")
  end = index
  if "key" in state:
    _append_plain(case, cache, "key", state["key"])
    _append_plain(case, cache, "value", state["value"])
    end = index + new
    fresh = ((slot >= index[:, None]) & (slot < end[:, None]))[:, None]
    if case["moved"]:
      where = slot + cache["dropped"].long()[:, None, None]
      cache["token_position"].copy_(torch.where(fresh, where.int(), cache["token_position"]))
      cache["token_weight"].masked_fill_(fresh, 0.0)
  values = lambda n: cache["cached_" + n].float() * (cache[n + "_absmax"] / 127).repeat_interleave(case["block"], 2)[..., None]  # noqa: E731
  query = q.float().view(b, new, kv, h // kv, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim)  # [B, Hk, group * new, D]
  s = (query @ values("key").transpose(2, 3)).view(b, kv, h // kv, new, room)
  at = index[:, None] + torch.arange(new, device="cuda")  # [B, new]
  if case["bias"]:
    here = cache["token_position"].long() if case["moved"] else slot.expand(b, kv, room)
    mine = at + (cache["dropped"].long()[:, None] if case["moved"] else 0)
    buckets = _bucket(mine[:, None, :, None] - here[:, :, None, :])  # [B, Hk, new, room]
    table = state["bias"].view(kv, h // kv, BUCKETS)
    s = s + torch.stack([t[torch.arange(kv, device="cuda")[:, None, None], buckets] for t in table.unbind(1)], 2)
  seen = (slot < end[:, None])[:, None].expand(b, new, room)
  if "key" in state:
    seen = seen & (slot <= at[:, :, None])
  if case["mask"]:
    seen = seen & state["mask"][:, None]
  seen = seen[:, None, None]
  s = s.masked_fill(~seen, -math.inf)
  top = s.amax(4, keepdim=True)
  p = torch.where(seen, torch.exp(s - top), torch.zeros_like(s))
  p = p / p.sum(4, keepdim=True).clamp(min=1e-30)
  o = p.view(b, kv, -1, room) @ values("value")
  if case["moved"]:
    cache["token_weight"] += p.sum((2, 3))
  out = o.view(b, kv, h // kv, new, dim).permute(0, 3, 1, 2, 4).reshape(b, new, h, dim).to(q.dtype)
  return {"out": out, **_held_values(cache, "key" in state)}


def _evict_plain(state):
  case, cache, out = state["case"], state["cache"], state["into"]
  b, h, room, dim, keep, block = (case[k] for k in ("batch", "kv_heads", "room", "dim", "keep", "block"))
  held = cache["cache_index"].long().clamp(max=room)[:, None, None]
  slot = torch.arange(room, device="cuda")
  w = torch.where(slot >= held - case["recent"], math.inf, cache["token_weight"])
  w = torch.where(slot < held, w, -math.inf)
  kept = torch.sort(w, dim=2, descending=True, stable=True).indices[..., :keep]
  kept = torch.where(kept < held, kept, room).sort(2).values
  there = kept < room
  source = kept.clamp(max=room - 1)
  blocks = -(-keep // block)
  grown = lambda x: torch.nn.functional.pad(x, (0, blocks * block - keep))  # noqa: E731
  for name in ("key", "value"):
    most = torch.where(there, cache[name + "_absmax"].gather(2, source // block), torch.zeros_like(w[..., :1]))
    after = grown(most).view(b, h, blocks, block).amax(3)
    each = after.repeat_interleave(block, 2)[..., :keep]
    c = cache["cached_" + name].gather(2, source[..., None].expand(-1, -1, -1, dim)).float()
    c = torch.where((most == each)[..., None], c, _round(most[..., None], c, each[..., None])).to(torch.int8)
    into = out["cached_" + name][:, :, :keep]
    into.copy_(torch.where(there[..., None], c, into))
    into = out[name + "_absmax"][:, :, :blocks]
    into.copy_(torch.where(grown(there.float()).view(b, h, blocks, block).amax(3) > 0, after, into))
  for name in ("token_weight", "token_position"):
    into = out[name][:, :, :keep]
    into.copy_(torch.where(there, cache[name].gather(2, source), into))
  left = cache["cache_index"].clamp(max=min(keep, room))
  out["cache_index"].copy_(left)
  out["dropped"].copy_(cache["dropped"] + cache["cache_index"] - left)
  return {"kept": torch.where(there, kept, -1).int(), **out}


def _linear_plain(state):
  x = state["x"].float()
  most = x.abs().amax(1, keepdim=True)
  codes = _round(x, 127, most).float()
  y = codes @ state["codes"][:, :x.shape[1]].float().t()  # (whole numbers)
  y = y * (most / 127) * (state["absmax"] / 127)
  if state["residual"] is not None:
    y = y + state["residual"].float()
  return y.to(state["x"].dtype)


def work(case):
  if case["op"] == "linear8":
    rows, k, n, size = case["rows"], case["in"], case["out"], 4 if case["dtype"] == "float32" else 2
    return {"bytes": rows * k * size + n * k + n * 4 + rows * n * size * (2 if case["residual"] else 1), "flops": 2 * rows * n * k}
  held = _held(case)
  kv, dim, block = case["kv_heads"], case["dim"], case["block"]
  if case["op"] == "evict":
    kept = sum(min(n, case["keep"]) for n in held)
    # weights of all that is held; codes, positions and weights of what is kept, read and written; which those are
    return {"bytes": kv * (4 * sum(held) + kept * (2 * (2 * dim + 8 + 8 / block) + 4)), "flops": 4 * kv * kept * dim}
  size, new = 4 if case["dtype"] == "float32" else 2, case["new"]
  appended = 0 if case["held"] == "all" else new
  tokens = sum(held) + appended * len(held)
  rows = case["batch"] * new
  moved = 8 * sum(held) + 4 * tokens if case["moved"] else 0  # weights read and written, positions read
  return {"bytes": kv * (tokens * (2 * dim + 8 / block) + moved) + rows * size * dim * (2 * case["heads"] + (2 * kv if appended else 0))
                   + rows // new * appended * 2 * kv * dim + (case["batch"] * case["room"] if case["mask"] else 0),
          "flops": 4 * case["heads"] * new * tokens * dim}


# ----------------------------------------------------------------------------
# In 64 bits, from the definitions
# ----------------------------------------------------------------------------
def exact(case, seed):
  state = prepare(case, seed)
  if case["op"] == "linear8":
    return _linear_exact(state)
  if case["op"] == "evict":
    return _evict_exact(state)
  return _attend_exact(state)


def _linear_exact(state):
  case, out = state["case"], []
  weight = state["codes"][:, :case["in"]].double()
  for x, r in zip(state["x"].split(512), state["residual"].split(512) if case["residual"] else [None] * case["rows"]):
    x = x.double()
    largest = x.abs().max(1, keepdim=True).values
    y = (127 * x / largest).round() @ weight.T * largest * state["absmax"].double() / 127 ** 2
    out.append((y if r is None else y + r).float())
  return torch.cat(out)


def _evict_exact(state):
  """(A choice and its copies: what is kept is compared whole, and the largest of each block in 64 bits.)"""
  case, cache, into = state["case"], state["cache"], state["into"]
  out = {k: v.clone() for k, v in into.items()}
  out["kept"] = torch.full((case["batch"], case["kv_heads"], case["keep"]), -1, dtype=torch.int32, device="cuda")
  for b, held in enumerate(_held(case)):
    recent = list(range(max(0, held - case["recent"]), held))
    n = min(held, case["keep"])
    weight = cache["token_weight"][b, :, :held - len(recent)].double()
    order = torch.argsort(-weight, dim=1, stable=True)[:, :n - len(recent)]
    last = torch.tensor(recent, dtype=torch.long, device="cuda").expand(case["kv_heads"], -1)
    kept = torch.cat([order, last], 1).sort(1).values[:, :n]
    out["kept"][b, :, :n] = kept.int()
    for name in ("token_weight", "token_position"):
      out[name][b, :, :n] = torch.take_along_dim(cache[name][b], kept, 1)
    for name in ("key", "value"):
      a = torch.take_along_dim(cache[name + "_absmax"][b].double(), kept // case["block"], 1)
      c = torch.take_along_dim(cache["cached_" + name][b].double(), kept[..., None], 1)
      for i, (pa, pc) in enumerate(zip(a.split(case["block"], 1), c.split(case["block"], 1))):
        most = pa.max(1, keepdim=True).values
        out[name + "_absmax"][b, :, i] = most[:, 0].float()
        at = i * case["block"]
        out["cached_" + name][b, :, at:at + pc.shape[1]] = (pc * pa[..., None] / most[..., None]).round().to(torch.int8)
    out["cache_index"][b] = n
    out["dropped"][b] = cache["dropped"][b] + held - n
  return out


def _attend_exact(state):
  case, cache = state["case"], state["cache"]
  fresh = "key" in state
  group, new, block, room = case["heads"] // case["kv_heads"], case["new"], case["block"], case["room"]
  if case["batch"] * case["kv_heads"] * new > 40000 or work(case)["flops"] > 3e11:
    return None
  out = torch.empty(state["query"].shape, dtype=torch.float32, device="cuda")
  held = {k: v.clone() for k, v in _held_values(cache, fresh).items()}
  back = [min(n, 16) + int(16 * math.log(n / 16) / math.log(8)) if n >= 16 else n for n in range(FAR)]
  buckets = torch.tensor([min(x, 31) for x in back] + [31], device="cuda")
  for b, start in enumerate(_held(case)):
    stop = start + new if fresh else start
    for h in range(case["kv_heads"]):
      kv = {}
      for name in ("key", "value"):
        a = cache[name + "_absmax"][b, h].double().clone()
        c = cache["cached_" + name][b, h].double()
        x = None
        if fresh:
          x = state[name][b, :, h].double()
          c = c.clone()
          for k in range(start // block, (stop - 1) // block + 1):
            lo, hi = max(start, k * block), min(stop, (k + 1) * block)
            most = max(float(a[k]) if start > k * block else 0.0, float(x[lo - start:hi - start].abs().max()))
            c[k * block:lo] = (c[k * block:lo] * a[k] / most).round() if most != float(a[k]) else c[k * block:lo]
            c[lo:hi] = (127 * x[lo - start:hi - start] / most).round()
            a[k] = most
          held[name + "_absmax"][b, h] = a.float()
          held["cached_" + name][b, h] = c.to(torch.int8)
        kv[name] = c[:stop] * a.repeat_interleave(block)[:stop, None] / 127
      q = state["query"][b, :, h * group:(h + 1) * group].double()  # [new, group, D]
      s = torch.einsum("lgd,kd->glk", q, kv["key"])
      at = start + torch.arange(new, device="cuda")
      place = torch.arange(stop, device="cuda")
      if case["moved"]:
        held["token_position"][b, h, start:stop] = (at + cache["dropped"][b]).int()
        place = held["token_position"][b, h, :stop].long()
        at = at + cache["dropped"][b].long()
      if case["bias"]:
        far = (at[:, None] - place).clamp(0, FAR)
        s = s + state["bias"][h * group:(h + 1) * group].double()[:, buckets[far]]
      hidden = torch.zeros(new, stop, dtype=torch.bool, device="cuda")
      if fresh:
        hidden |= torch.arange(stop, device="cuda") > start + torch.arange(new, device="cuda")[:, None]
      if case["mask"]:
        hidden |= ~state["mask"][b, :stop]
      p = torch.softmax(s.masked_fill(hidden, -math.inf), 2).masked_fill(hidden, 0.0)
      out[b, :, h * group:(h + 1) * group] = torch.einsum("glk,kd->lgd", p, kv["value"]).float()
      if case["moved"]:
        w = held["token_weight"][b, h]
        w[start:stop] = 0
        w[:stop] = (w[:stop].double() + p.sum((0, 1))).float()
  return {"out": out, **held}
