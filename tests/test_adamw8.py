"""AdamW with moments in 8 bits, by tensor operations (what runs on the CPU and states what the kernel computes):
the rounding against its definition, what it does to a moment over many steps, states and refusals."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from t5x_b200 import optax_api, optimizers

# every finite e4m3 magnitude, in order
LEVELS = [Fraction(m, 8) * Fraction(2) ** -6 for m in range(8)] + \
    [(1 + Fraction(m, 8)) * Fraction(2) ** e for e in range(-6, 9) for m in range(8)][:-1]


def test_levels():
  got = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().tolist()
  assert [Fraction(v) for v in got] == LEVELS and LEVELS[-1] == 448


def rounded(y: Fraction, noise: int) -> int:
  """The code of y in [0, 448]: the upper neighbour where (y - lower) / (upper - lower) + (noise + 1/2) / 2^16
  reaches 1."""
  low = max(i for i, v in enumerate(LEVELS) if v <= y)
  if LEVELS[low] == y or low == 126:
    return low
  part = (y - LEVELS[low]) / (LEVELS[low + 1] - LEVELS[low])
  return low + (part + Fraction(2 * noise + 1, 1 << 17) >= 1)


@pytest.mark.parametrize("second", [False, True])
@pytest.mark.parametrize("size", [1, 5, 255, 256, 257, 700])
@pytest.mark.parametrize("scale", [1.0, 1e-36, 1e36])
def test_rounding(second, size, scale):
  gen = torch.Generator().manual_seed(size)
  x = torch.randn(size, generator=gen) * torch.exp(4 * torch.randn(size, generator=gen))
  x = x.clamp(-100, 100) * scale
  if second:
    x = x.abs()
  x[:: 7] = 0
  noise = optimizers._moment_noise(size, 3, 9, "cpu") & 0xFFFF
  codes, absmax = optimizers.quantize_moment(x, noise, second)
  assert codes.shape == x.shape and absmax.shape == (-(-size // 256),)
  for i in range(size):
    most = x[i // 256 * 256: i // 256 * 256 + 256].abs().max()
    assert absmax[i // 256] == most
    code, v = int(codes[i]), float(x[i])
    if most == 0:
      assert code & 127 == 0
      continue
    # y is computed in 32 bits with three roundings, 2^-24 each; the noise then moves by at most that part of a step,
    # so the exact y moved by as much to either side has to give the code on one of them
    y = Fraction(abs(v)) / Fraction(float(most)) * 448
    around = [rounded(min(y * (1 + Fraction(s, 1 << 22)), Fraction(448)), int(noise[i])) for s in (-1, 0, 1)]
    if second and v > 0:
      around = [max(1, c) for c in around]
    assert code & 127 in around
    assert (code >> 7) == (0 if second or v >= 0 else 1) or code & 127 == 0
  back = optimizers.dequantize_moment(codes, absmax)
  assert torch.all((back > 0) == (x > 0)) if second else torch.all(back * x >= 0)


def test_noise():
  """The hash against arithmetic modulo 2^32 on Python's integers; 16-bit halves spread evenly."""
  n, seed, step = 1 << 16, 11, 1234
  h = optimizers._moment_noise(n, seed, step, "cpu")
  for i in (0, 1, 2, 255, 256, 65535):
    v = (i + seed * 0x9E3779B1 + step * 0xBB67AE85) % 2 ** 32
    for factor, shift in ((0x9E3779B1, 15), (0x6A09E667, 13), (0xBB67AE85, 16)):
      v = v * factor % 2 ** 32
      v ^= v >> shift
    assert int(h[i]) == v
  for half in (h & 0xFFFF, h >> 16):
    counts = np.bincount((half >> 8).numpy(), minlength=256)
    chi2 = ((counts - n / 256) ** 2 / (n / 256)).sum()
    assert abs(chi2 - 255) < 6 * math.sqrt(2 * 255)  # 255 degrees of freedom, variance twice that


def test_second_moment_follows_the_gradients():
  """A gradient of constant size s after 3000 steps with b2 = 0.999: nu = s^2 (1 - 0.999^3000) = 0.950 s^2. Rounded
  to the nearest code, it would stop where 0.001 s^2 is half a step."""
  n, steps, b2 = 4096, 3000, 0.999
  gen = torch.Generator().manual_seed(0)
  sizes = torch.exp(torch.randn(n, generator=gen) * 0.5)
  t = optimizers.scale_by_adam8(b2=b2)
  state = t.init({"w": sizes})
  for i in range(steps):
    _, state = t.update({"w": sizes}, state)
  got = optimizers.dequantize_moment(state["nu"]["w"], state["nu_absmax"]["w"])
  ratio = got / sizes.square() / (1 - b2 ** steps)
  # the mean is kept; one value's spread: a jump is at most 1/8 of the value up or down and the jumps of a thousand
  # steps are summed, with probability 0.001 / (1/16) each: variance below 2 * 0.016 * 1000 * (1/8)^2 / 2 = 0.25
  assert abs(float(ratio.mean()) - 1) < 6 * 0.5 / math.sqrt(n)
  assert float(ratio.std()) < 0.5


@pytest.mark.parametrize("shape", [(3, 5), (256,), (17, 31), (0,), ()])
def test_first_step_against_64_bits(shape):
  gen = torch.Generator().manual_seed(1)
  w = torch.randn(shape, generator=gen)
  g = torch.randn(shape, generator=gen)
  lr, eps, wd = 0.01, 1e-8, 0.1
  opt = optimizers.adamw8(lr, eps=eps, weight_decay=wd).create({"a": {"w": w.clone()}})
  new = opt.apply_gradient({"a": {"w": g}})
  gd, wd64 = g.double(), w.double()
  m, v = 0.1 * gd, 0.001 * gd ** 2  # (the factors 1 - b cancel against the bias corrections, to 32 bits)
  want = wd64 - lr * ((m / 0.1) / ((v / 0.001).sqrt() + eps) + wd * wd64)
  assert torch.allclose(new.target["a"]["w"].double(), want, rtol=0, atol=1e-6)
  adam = new.state.param_states["0"]
  assert int(adam["count"]) == 1 and adam["mu"]["a"]["w"].shape == w.shape
  # e4m3 rounds by less than one step: an eighth of the value, or 2^-9 / 448 of the largest of the block
  for name, x in (("mu", m), ("nu", v)):
    got = optimizers.dequantize_moment(adam[name]["a"]["w"], adam[name + "_absmax"]["a"]["w"]).double()
    if x.numel():
      assert torch.all((got - x).abs() <= x.abs() / 8 + x.abs().max() / (448 * 512) * 1.001)


def test_state_layout_axes_and_restore(tmp_path):
  from t5x_b200 import checkpoints, partitioning, train_state
  definition = optimizers.chain([optimizers.clip_by_global_norm(1.0), optax_api.adamw8(1e-2)])
  assert definition.fused_plan is None and definition.fused_plan8["bits"] == 8
  gen = torch.Generator().manual_seed(2)
  variables = lambda: {"params": {"l": {"kernel": torch.randn(6, 50, generator=gen), "scale": torch.ones(7)}},  # noqa: E731
                       "params_axes": {"l": {"kernel": ("embed", "mlp"), "scale": ("embed",)}}}
  state = train_state.FlaxOptimTrainState.create(definition, variables())
  grads = {"l": {"kernel": torch.randn(6, 50, generator=gen), "scale": torch.randn(7, generator=gen)}}
  state = state.apply_gradient(grads, learning_rate=None)
  axes = state.as_logical_axes().param_states["1"]["0"]
  assert axes["mu"]["l"]["kernel"] == ("embed", "mlp") and axes["mu_absmax"]["l"]["kernel"] == (None,)
  adam = state.param_states["1"]["0"]
  assert adam["nu"]["l"]["kernel"].dtype == torch.uint8 and adam["nu_absmax"]["l"]["kernel"].shape == (2,)

  partitioner = partitioning.PjitPartitioner(num_partitions=1)
  saver = checkpoints.Checkpointer(state, partitioner, str(tmp_path))
  saver.save(state)
  fresh = train_state.FlaxOptimTrainState.create(definition, variables())
  back = checkpoints.Checkpointer(fresh, partitioner, str(tmp_path)).restore()
  for name in ("mu", "nu", "mu_absmax", "nu_absmax"):
    for leaf in ("kernel", "scale"):
      got, want = back.param_states["1"]["0"][name]["l"][leaf], adam[name]["l"][leaf]
      assert got.dtype == want.dtype and torch.equal(got, want), name
  a, b = back.apply_gradient(grads, None), state.apply_gradient(grads, None)
  assert torch.equal(a.params["l"]["kernel"], b.params["l"]["kernel"])


def test_refused_under_a_model_or_expert_axis():
  from t5x_b200.parallel import state as pstate
  st = pstate.get()
  for name in ("model_size", "expert_size"):
    setattr(st, name, 2)
    try:
      with pytest.raises(ValueError, match="whole parameters"):
        optimizers.adamw8(1e-3).create({"w": torch.zeros(4)})
    finally:
      setattr(st, name, 1)


def test_decay_mask_takes_the_general_path():
  definition = optimizers.adamw8(0.1, weight_decay=0.5, mask={"w": True, "b": False})
  assert definition.fused_plan is None and definition.fused_plan8 is None
  p = {"w": torch.ones(3), "b": torch.ones(3)}
  new = definition.create(p).apply_gradient({"w": torch.zeros(3), "b": torch.zeros(3)})
  assert torch.allclose(new.target["w"], torch.full((3,), 0.95)) and torch.equal(new.target["b"], torch.ones(3))


def test_earlier_optimizer_keeps_its_count():
  opt = optimizers.adamw8(0.1).create({"a": {"w": torch.ones(3)}})
  new = opt.apply_gradient({"a": {"w": torch.ones(3)}})
  assert int(opt.state.param_states["0"]["count"]) == 0 and int(new.state.param_states["0"]["count"]) == 1


# ---- refusals of the C entry points, with made-up addresses: nothing is launched ----
A = 1 << 20


def _item(**kw):
  import struct
  f = dict(p=A, g=A, mu=A, nu=A, out=A, mu_absmax=A, nu_absmax=A, n=10)
  f.update(kw)
  return ctypes.create_string_buffer(struct.pack("=7Qq", *[f[k] for k in
                                                           ("p", "g", "mu", "nu", "out", "mu_absmax", "nu_absmax", "n")]))


@pytest.mark.parametrize("bits,item,message", [
    (32, dict(p=0), "null"), (32, dict(g=0), "null"), (8, dict(mu_absmax=0), "null"), (8, dict(nu_absmax=0), "null"),
    (32, dict(p=A + 2), "misaligned"), (32, dict(mu=A + 1), "misaligned"), (8, dict(nu_absmax=A + 2), "misaligned"),
    (32, dict(out=A + 1), "misaligned"), (32, dict(n=-1), "negative"), (16, {}, "8 or 32"), (32, dict(n=1 << 42), "large")])
def test_step_refusals(bits, item, message):
  from t5x_b200.ops import native
  lib, buf = native.lib(), _item(**item)
  assert lib.t5x_adamw_group(ctypes.addressof(buf), 1, bits, 0.1, 0.9, 0.99, 1e-8, 0.0, 0.0, 1, 0, None, None) != 0
  assert message in lib.t5x_last_error().decode()


def test_other_refusals():
  from t5x_b200.ops import native
  lib, buf = native.lib(), _item()
  at = ctypes.addressof(buf)
  assert lib.t5x_adamw_group(at, 1, 32, 0.1, 0.9, 0.99, 1e-8, 0.0, 0.0, 0, 0, None, None) != 0
  assert "from 1" in lib.t5x_last_error().decode()
  assert lib.t5x_adamw_group(None, 1, 32, 0.1, 0.9, 0.99, 1e-8, 0.0, 0.0, 1, 0, None, None) != 0
  assert lib.t5x_grad_clip_scale(at, 1, None, 1.0, A, None) != 0
  assert lib.t5x_grad_clip_scale(at, 1, A + 4, 1.0, A, None) != 0
  assert "misaligned" in lib.t5x_last_error().decode()
  items = native.AdamwItems()
  w, mu, nu, few = torch.zeros(300), torch.zeros(300), torch.zeros(300), torch.zeros(2, 10)
  with pytest.raises(native.NativeError, match="types and sizes"):
    items.add(w, w, torch.zeros(300, dtype=torch.uint8), torch.zeros(300, dtype=torch.uint8), None,
              torch.zeros(1), torch.zeros(2))
  items.add(w, w, mu, nu)
  assert not items.overlap()
  items.add(w[10:20], w[:10], few[0], few[1])
  assert items.overlap()
