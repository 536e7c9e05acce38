"""Decoding in 8 bits as the models reach it: `kv_cache_dtype`, `kv_cache_keep`, `layers.quantize_dense`."""
import copy

import numpy as np
import pytest
import torch

from t5x_b200 import adafactor
from t5x_b200 import decoding
from t5x_b200 import decoding_fast
from t5x_b200 import models
from t5x_b200 import optax_api
from t5x_b200 import optimizers
from t5x_b200.data import vocabularies
from t5x_b200.models.decoder_only import network as decoder_only
from t5x_b200.models.t5 import layers
from t5x_b200.models.t5 import network as t5
from t5x_b200.ops import cache8
from t5x_b200.ops import functional as F
from t5x_b200.ops import native

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def attention_layer(device, **kw):
  torch.manual_seed(0)
  dtype = "bfloat16" if device == "cuda" else "float32"
  attn = layers.MultiHeadDotProductAttention(64, 2, 64 if device == "cuda" else 8, dtype, kv_cache_dtype="int8", **kw)
  return attn.to(device), torch.randn(2, 32).to(device) * 0.3  # (heads, buckets)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("keep", [0, 20])
@torch.no_grad()
def test_a_layer_decodes_as_the_operators_do(device, keep):
  """A prompt, then tokens one at a time past two evictions: the layer's results are those of the operators called in turn."""
  attn, table = attention_layer(device, kv_cache_keep=keep, kv_cache_recent=5 if keep else 0)
  lengths = torch.tensor([30, 11], device=device)
  max_len, lk, steps = 250, 30, 140
  cache = attn.init_cache(2, max_len, device)
  assert ("cache_room" in cache) == bool(keep) and cache["cached_key"].shape[2] == (96 if keep else 256)
  kw = dict(bias_table=table, bidirectional=False)
  prompt = torch.randn(2, lk, 64, device=device).to(attn.dtype)
  attn(prompt, prompt, cache=cache, prefill=True, prefill_lengths=lengths, causal=True, **kw)

  heads = lambda x: x.view(2, -1, 2, attn.head_dim)  # noqa: E731
  q, k, v = (heads(m(prompt)) for m in (attn.query, attn.key, attn.value))
  mine = cache8.init_cache(2, 32 if keep else max_len, 2, attn.head_dim, device, weights=bool(keep), positions=bool(keep))
  cache8.append_(mine, k, v, lengths)
  mine["cache_index"] += lengths.int()
  room = None
  if keep:
    # the last 30 queries of each row (of the shorter one 11, behind 19 that see nothing)
    last = torch.stack([q[0], torch.cat([q[1, :1].expand(19, -1, -1), q[1, :11]])])
    cache8.attention(last, mine, bias_table=table)
    mine, _ = cache8.evict(mine, keep, recent=5, out=cache8.init_cache(2, 96, 2, attn.head_dim, device, weights=True, positions=True))
    room = 64
  before = native.launch_count() if device == "cuda" else 0
  for i in range(steps):
    x = torch.randn(2, 1, 64, device=device).to(attn.dtype)
    got = attn(x, x, cache=cache, decode=True, **kw)
    if room == 0:
      mine, _ = cache8.evict(mine, keep, recent=5)
      room = 64
    want = cache8.attention(heads(attn.query(x)), mine, heads(attn.key(x)), heads(attn.value(x)), bias_table=table)
    mine["cache_index"] += 1
    if keep:
      room -= 1
    # (the layer's three projections may be one product: as near as roundings of the type are)
    assert torch.allclose(got, attn.out(want.reshape(2, 1, -1)), rtol=0.03, atol=0.03 if device == "cuda" else 1e-5)
    if device == "cpu":
      assert all(torch.equal(cache[n].expand(mine[n].shape), mine[n]) for n in mine if n != "token_weight")
  if keep:
    assert cache["cache_index"].max() <= 84 and cache["dropped"].tolist() == (lengths + steps - cache["cache_index"]).tolist()
  assert device == "cpu" or native.launch_count() > before


def decoder_only_model(device, **kw):
  torch.manual_seed(0)
  cfg = decoder_only.TransformerConfig(vocab_size=32, emb_dim=64, num_heads=2, head_dim=64 if device == "cuda" else 8, mlp_dim=64,
                                       num_layers=2, dropout_rate=0.0, mlp_activations=("gelu", "linear"),
                                       dtype="bfloat16" if device == "cuda" else "float32", **kw)
  return models.DecoderOnlyModel(decoder_only.DecoderWrapper(cfg).to(device), vocabularies.PassThroughVocabulary(32),
                                 adafactor.Adafactor(), inputs_bidirectional_attention=False)


@pytest.mark.parametrize("device", DEVICES)
def test_a_decoder_only_model_generates(device):
  tokens = torch.randint(2, 32, (3, 150), generator=torch.Generator().manual_seed(0)).to(device)
  seen = torch.zeros(3, 150, dtype=torch.long, device=device)
  seen[0, :40], seen[1, :7], seen[2, :100] = 1, 1, 1
  batch = {"decoder_input_tokens": torch.cat([tokens[:, :1] * 0, tokens[:, 1:]], 1), "decoder_causal_attention": seen}
  out = {}
  for name, kw in (("plain", {}), ("int8", dict(kv_cache_dtype="int8")),
                   ("all", dict(kv_cache_dtype="int8", kv_cache_keep=140, kv_cache_recent=1)),
                   ("some", dict(kv_cache_dtype="int8", kv_cache_keep=16, kv_cache_recent=4))):
    model = decoder_only_model(device, **kw)
    model._decode_fn = lambda **kw: decoding.temperature_sample(topk=1, **kw)
    out[name] = model.predict_batch(None, batch, rng=None)
  assert out["int8"].shape == out["plain"].shape == out["some"].shape
  assert torch.equal(torch.as_tensor(out["int8"]), torch.as_tensor(out["all"]))


@pytest.mark.parametrize("device", DEVICES)
def test_an_encoder_decoder_decodes(device):
  """Beam search and sampling: cross attention's keys in 8 bits are projected once and shared by the beams."""
  torch.manual_seed(1)
  cfg = dict(vocab_size=64, emb_dim=64, num_heads=2, head_dim=64 if device == "cuda" else 8, mlp_dim=64, num_encoder_layers=1,
             num_decoder_layers=2, dropout_rate=0.0, mlp_activations=("gelu", "linear"),
             dtype="bfloat16" if device == "cuda" else "float32")
  vocab = vocabularies.PassThroughVocabulary(64)
  x = torch.randint(2, 64, (3, 20), generator=torch.Generator().manual_seed(2)).to(device)
  x[0, 12:] = 0
  batch = {"encoder_input_tokens": x, "decoder_input_tokens": torch.zeros(3, 15, dtype=torch.long, device=device)}
  for fn in (decoding.beam_search, decoding.temperature_sample):
    module = t5.Transformer(t5.T5Config(**cfg, kv_cache_dtype="int8")).to(device)
    assert not decoding_fast.supported(module, batch["decoder_input_tokens"], fn)
    model = models.EncoderDecoderModel(module, vocab, vocab, adafactor.Adafactor(), decode_fn=fn)
    out, aux = model.predict_batch_with_aux(None, batch, num_decodes=2, return_all_decodes=True)
    assert out.shape == (3, 2, 15) and np.isfinite(np.asarray(torch.as_tensor(aux["scores"]).cpu())).all()


@pytest.mark.parametrize("device", DEVICES)
def test_quantized_projections(device):
  model = decoder_only_model(device)
  module = model.module
  ids = torch.randint(2, 32, (2, 9)).to(device)
  with torch.no_grad():
    plain = module(ids, ids, enable_dropout=False)
    dense = module.decoder.layers_0.mlp.wi_0
    x = torch.randn(3, 5, 64, device=device).to(dense.dtype)
    want = F.linear8(x, F.quantize_weight(dense.kernel))
    assert layers.quantize_dense(module) == 2 * 7
    assert torch.equal(dense(x), want)
    quantized = module(ids, ids, enable_dropout=False)
    assert quantized.shape == plain.shape and not torch.equal(quantized, plain)
    dense.kernel.add_(1.0)
    with pytest.raises(ValueError, match="quantize_dense"):
      dense(x)
    layers.quantize_dense(module)
    assert torch.equal(dense(x), F.linear8(x, F.quantize_weight(dense.kernel)))
    dense.kernel.sub_(1.0)
    layers.dequantize_dense(module)
    assert torch.allclose(module(ids, ids, enable_dropout=False), plain, rtol=1e-2, atol=1e-2)
  layers.quantize_dense(module)
  with pytest.raises(ValueError, match="no_grad"):
    module(ids, ids, enable_dropout=False)


def test_refusals():
  for kw in (dict(kv_cache_dtype="int4"), dict(kv_cache_keep=8), dict(kv_cache_dtype="int8", kv_cache_keep=8, kv_cache_recent=9)):
    with pytest.raises(ValueError):
      layers.MultiHeadDotProductAttention(16, 2, 8, **kw)
  attn, table = attention_layer("cpu")
  cache = attn.init_cache(2, 16, "cpu")
  x = torch.randn(2, 1, 64)
  with pytest.raises(ValueError, match="no_grad"):
    attn(x, x, cache=cache, decode=True, bidirectional=False)
  with pytest.raises(ValueError, match="causal"), torch.no_grad():
    attn(x, x, cache=cache, decode=True, bias_table=table)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("steps", [[100], [30, 64, 7, 130, 1], [65, 65]])
@torch.no_grad()
def test_steps_of_more_tokens_than_an_eviction_makes_room_for(device, steps):
  """No token is left out: the cache and the results are those of parts of 64 tokens, given one after the other."""
  attn, table = attention_layer(device, kv_cache_keep=20, kv_cache_recent=5)
  x = (torch.randn(2, sum(steps), 64, device=device) / 4).to(attn.dtype)
  kw = dict(bias_table=table, bidirectional=False, decode=True)
  outs = []
  for sizes in (steps, [n for step in steps for n in [64] * (step // 64) + [step % 64] if n]):
    cache = attn.init_cache(2, 400, device)
    outs.append((torch.cat([attn(p, p, cache=cache, **kw) for p in x.split(sizes, 1)], 1), cache))
    assert 0 <= cache["cache_room"] <= 96 and cache["cache_index"].max() <= 84
    held = cache["cache_index"].expand(2) + (cache["dropped"] if "dropped" in cache else 0)
    assert held.tolist() == [sum(steps)] * 2
  (got, one), (want, other) = outs
  # (the projections of parts may round the other way)
  assert torch.allclose(got, want, rtol=0.03, atol=0.03 if device == "cuda" else 1e-5)
  assert one["cache_room"] == other["cache_room"] and one["dropped"].tolist() == other["dropped"].tolist()


STEPS = {"adafactor": lambda: adafactor.Adafactor(min_dim_size_to_factor=0),
         "adafactor of vectors": lambda: adafactor.Adafactor(min_dim_size_to_factor=1000),
         "adamw": lambda: optimizers.adamw(0.1),
         "clipped adamw": lambda: optimizers.chain([optimizers.clip_by_global_norm(0.5), optax_api.adamw(0.1)]),
         "adamw8": lambda: optimizers.adamw8(0.1), "sgd": lambda: optimizers.sgd(0.1)}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", STEPS)
def test_a_step_of_an_optimizer_is_seen_by_quantized_projections(device, name):
  """Its kernels write the parameters through pointers, its statements through `.data`."""
  torch.manual_seed(0)
  dense = layers.DenseGeneral(64, 96, ("embed", "mlp"), device=device)
  layers.quantize_dense(dense)
  x = torch.randn(3, 64, device=device)
  before = dense.kernel.detach().clone()
  with torch.no_grad():
    stale = dense(x)
  optimizer = STEPS[name]().create({"mlp": {"kernel": dense.kernel}})
  optimizer.apply_gradient({"mlp": {"kernel": torch.randn(64, 96, device=device)}}, learning_rate=0.1)
  assert not torch.equal(dense.kernel, before)
  with torch.no_grad():
    with pytest.raises(ValueError, match="quantize_dense"):
      dense(x)
    layers.quantize_dense(dense)
    assert torch.equal(dense(x), F.linear8(x, F.quantize_weight(dense.kernel))) and not torch.equal(dense(x), stale)


def test_copies_of_quantized_projections_and_kernels_of_inference_mode():
  torch.manual_seed(0)
  dense = layers.DenseGeneral(64, 96, ("embed", "mlp"))
  x = torch.randn(3, 64)
  with torch.no_grad():
    dense.kernel.mul_(2.0)
    layers.quantize_dense(dense)
    twin = copy.deepcopy(dense)
    assert torch.equal(twin(x), dense(x))
    twin.kernel.add_(1.0)
    with pytest.raises(ValueError, match="quantize_dense"):
      twin(x)
    dense(x)
    with pytest.raises(ValueError, match="quantize_dense"):
      copy.deepcopy(twin)(x)
    dense.kernel = torch.nn.Parameter(dense.kernel.clone())
    with pytest.raises(ValueError, match="quantize_dense"):
      dense(x)
  with torch.inference_mode():
    dense = layers.DenseGeneral(64, 96, ("embed", "mlp"))
    layers.quantize_dense(dense)
    assert torch.equal(dense(x), F.linear8(x, F.quantize_weight(dense.kernel)))


def test_a_quantized_projection_under_grad_mode():
  """Its kernel would get no gradient: refused, where the kernel wants one."""
  dense = layers.DenseGeneral(64, 96, ("embed", "mlp"))
  layers.quantize_dense(dense)
  x = torch.randn(3, 64)
  with pytest.raises(ValueError, match="no_grad"):
    dense(x)
  with torch.no_grad():
    want = dense(x)
  with torch.inference_mode():
    assert torch.equal(dense(x), want)
  dense.kernel.requires_grad_(False)
  assert torch.equal(dense(x), want)
  with pytest.raises(ValueError, match="no_grad"):
    dense(x.requires_grad_())


@pytest.mark.parametrize("name", ["query", "key", "value", "out", "wi_0", "wi_1", "wo"])
@torch.no_grad()
def test_a_projection_quantized_by_itself(name):
  """It multiplies in 8 bits where its layer runs, whatever the projections beside it do."""
  torch.manual_seed(0)
  attn = layers.MultiHeadDotProductAttention(64, 2, 8, "float32")
  mlp = layers.MlpBlock(64, 32, ("gelu", "linear"), 0.0, "float32")
  x = torch.randn(2, 5, 64)
  run = lambda: (attn(x, x), mlp(x))  # noqa: E731
  plain = run()
  module = getattr(attn, name, None) or getattr(mlp, name)
  assert layers.quantize_dense(module) == 1
  calls, forward = [], F.linear8
  F.linear8 = lambda *args, **kw: (calls.append(args[1]), forward(*args, **kw))[1]
  try:
    got = run()
  finally:
    F.linear8 = forward
  assert len(calls) == 1 and calls[0] is module.weight8.codes
  assert [torch.equal(a, b) for a, b in zip(got, plain)] == [hasattr(mlp, name), hasattr(attn, name)]


@torch.no_grad()
def test_masks_and_biases_that_a_cache_in_8_bits_does_not_take():
  attn, table = attention_layer("cpu")
  x, ids = torch.randn(2, 1, 64), torch.ones(2, 1, dtype=torch.long)
  run = lambda **kw: attn(x, x, cache=attn.init_cache(2, 16, "cpu"), decode=True, bidirectional=False, **kw)  # noqa: E731
  run(bias_table=table)
  cross = attn.cross_cache(torch.randn(2, 7, 64))
  over = lambda **kw: attn(x, None, precomputed_kv=cross, **kw)  # noqa: E731
  over(key_mask=torch.ones(2, 7, dtype=torch.bool))
  for kw in (dict(extra_mask=torch.ones(2, 1, 1, 1)), dict(explicit_bias=torch.ones(1, 2, 1, 1)), dict(q_segment_ids=ids),
             dict(kv_segment_ids=ids)):
    for call in (run, over):
      with pytest.raises(ValueError, match=next(iter(kw))):
        call(**kw)
  for call in (lambda: run(key_mask=torch.ones(2, 16, dtype=torch.bool)), lambda: over(bias_table=table), lambda: over(causal=True)):
    with pytest.raises(ValueError, match="8 bits"):
      call()
