"""AdamW over many parameters in one launch, moments in 32 and in 8 bits: against 64 bits, against the kernel of one
parameter, against the tensor operations that state it, and the calls that it has to leave to another path."""
import math

import pytest
import torch

from t5x_b200 import optimizers

pytestmark = pytest.mark.gpu

SIZES = [1, 2, 3, 255, 256, 257, 1023, 2047, 2048, 2049, 4096, 70001, 0, 12, 300000]


def tree(sizes, seed, offset=0, bf16=True, scale=1.0):
  """{"part<i>": {"w<i>": tensor}}; offset: values that the tensor starts behind an aligned address."""
  gen = torch.Generator(device="cuda").manual_seed(seed)
  out = {}
  for i, n in enumerate(sizes):
    t = (torch.randn(n + offset, device="cuda", generator=gen) * scale)[offset:]
    if bf16 and i % 3 != 2:
      t.bf16 = torch.empty(n + offset, dtype=torch.bfloat16, device="cuda")[offset:]
    out.setdefault("part%d" % (i % 4), {})["w%d" % i] = t
  return out


def leaves(t):
  return [v for _, v in sorted(optimizers.flatten(t).items())]


def adam_of(opt):
  def find(node):
    return node if "mu" in node else next((f for f in map(find, (v for v in node.values() if isinstance(v, dict)))
                                           if f is not None), None)
  return find(opt.state.param_states)


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_32_bits_match_the_kernel_of_one_parameter(offset, wd):
  """The same expressions in the same order: bit for bit, over three steps."""
  from t5x_b200.ops import comm, native
  grads = [tree(SIZES, 10 + s, offset, bf16=False) for s in range(3)]
  got = optimizers.adamw(3e-3, weight_decay=wd).create(tree(SIZES, 1, offset))
  want = tree(SIZES, 1, offset)
  mus = [torch.zeros_like(p) for p in leaves(want)]
  nus = [torch.zeros_like(p) for p in leaves(want)]
  for step, g in enumerate(grads):
    before = native.launch_count()
    got = got.apply_gradient(g)
    assert native.launch_count() - before == 1
    for p, gg, m, v in zip(leaves(want), leaves(g), mus, nus):
      bf = getattr(p, "bf16", None)
      native.adamw_step_(p, gg, m, v, comm._ptr_array([] if bf is None else [bf.data_ptr()]), 0, lr=3e-3, b1=0.9,
                         b2=0.999, eps=1e-8, eps_root=0.0, weight_decay=wd, step=step + 1, clip_scale=None)
  adam = adam_of(got)
  for a, b, m, v, gm, gv in zip(leaves(got.target), leaves(want), mus, nus, leaves(adam["mu"]), leaves(adam["nu"])):
    assert torch.equal(a, b) and torch.equal(m, gm) and torch.equal(v, gv)
    if getattr(b, "bf16", None) is not None:
      assert torch.equal(a.bf16, b.bf16) and torch.equal(a.bf16, a.to(torch.bfloat16))
  native.check_status()


def reference_step(p, g, mu, nu, step, lr, wd, factor=1.0, b1=0.9, b2=0.999, eps=1e-8):
  """In 64 bits."""
  p, g, mu, nu = (t.double() for t in (p, g, mu, nu))
  g = g * factor
  mu, nu = b1 * mu + (1 - b1) * g, b2 * nu + (1 - b2) * g * g
  u = (mu / (1 - b1 ** step)) / ((nu / (1 - b2 ** step)).sqrt() + eps) + wd * p
  return p - lr * u, mu, nu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("host", ["1", "0"])
def test_many_tensors_against_64_bits(bits, host, monkeypatch):
  """More tensors than one launch takes."""
  from t5x_b200.ops import native
  monkeypatch.setattr(native, "_host", None if host == "1" else False)
  sizes = [1 + (37 * i) % 600 for i in range(1000)]
  make = optimizers.adamw if bits == 32 else optimizers.adamw8
  lr, wd = 1e-2, 0.05
  opt = make(lr, weight_decay=wd).create(tree(sizes, 3))
  g = tree(sizes, 4, bf16=False)
  before = [p.clone() for p in leaves(opt.target)]
  count = native.launch_count()
  opt = opt.apply_gradient(g)
  assert native.launch_count() - count == (2 if bits == 32 else 3)  # 576 or 448 a launch
  zero = torch.zeros((), device="cuda")
  for p, p0, gg in zip(leaves(opt.target), before, leaves(g)):
    want, _, _ = reference_step(p0, gg, zero, zero, 1, lr, wd)
    # a dozen roundings of 2^-24 in an update of about lr, the approximate root and quotients 2^-22 each
    assert torch.all((p.double() - want).abs() <= lr * 2 ** -19 + p0.abs() * 2 ** -23)
    if getattr(p, "bf16", None) is not None:
      assert torch.equal(p.bf16, p.to(torch.bfloat16))


def to_cpu(t):
  return {k: to_cpu(v) if isinstance(v, dict) else v.cpu() for k, v in t.items()}


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_8_bits_match_the_tensor_operations(offset, max_norm):
  """Three steps on the GPU, each from the same state as a step of the generic chain on the CPU. The update and the
  scales agree to 32 bits; a code may be that of the next number where the draw falls beside its border: the value
  before rounding differs by some 2^-21 of itself between the two, a step is 2^-4 of it or more, so the draws that
  this moves are some 2^-16 of all: 10 of these 380,000 on average (and only to a neighbour)."""
  def chain():
    parts = [optimizers.clip_by_global_norm(max_norm)] if max_norm else []
    return optimizers.chain(parts + [optimizers._adamw8(1e-2, weight_decay=0.1, seed=5)])

  gpu = chain().create(tree(SIZES, 1, offset))
  for step in range(3):
    g = tree(SIZES, 20 + step, offset, bf16=False, scale=10.0 ** (step - 2))
    cpu = chain().create(to_cpu(gpu.target))
    cpu.state.param_states = to_cpu(gpu.state.param_states)
    gpu, cpu = gpu.apply_gradient(g), cpu.apply_gradient(to_cpu(g))
    for p, q in zip(leaves(gpu.target), leaves(cpu.target)):
      assert torch.allclose(p.cpu(), q, rtol=2 ** -22, atol=1e-2 * 2 ** -18)
      if getattr(p, "bf16", None) is not None:
        assert torch.equal(p.bf16, p.to(torch.bfloat16))
    a, b = adam_of(gpu), adam_of(cpu)
    assert int(a["count"]) == int(b["count"]) == step + 1
    off = 0
    for name in ("mu", "nu"):
      for x, y in zip(leaves(a[name + "_absmax"]), leaves(b[name + "_absmax"])):
        # without a clip half a dozen roundings of 2^-24. The chain's norm is a sum of 32-bit squares: 19 levels of
        # pairs over 400,000 values and 15 tensors in turn, 34 * 2^-24, half of it in the root and all of it again
        # in the square of the factor, 2^-19 with the others
        assert torch.allclose(x.cpu(), y, rtol=2 ** -18 if max_norm else 2 ** -20, atol=0)
      for x, y in zip(leaves(a[name]), leaves(b[name])):
        d = (x.cpu().int() - y.int()).abs()
        assert d.numel() == 0 or int(d.max()) <= 1
        off += int((d > 0).sum())
    assert off < 60


@pytest.mark.parametrize("bits", [32, 8])
def test_host_path_and_its_stand_in_agree(bits, monkeypatch):
  from t5x_b200.ops import native

  def run():
    make = optimizers._adamw if bits == 32 else optimizers._adamw8
    clip = [optimizers.clip_by_global_norm(0.3)]
    opt = optimizers.chain(clip + [make(1e-2)]).create(tree(SIZES, 1))
    for s in range(2):
      opt = opt.apply_gradient(tree(SIZES, 5 + s, bf16=False))
    return leaves(opt.target) + leaves(adam_of(opt)["mu"]) + leaves(adam_of(opt)["nu"])

  with_host = run()
  monkeypatch.setattr(native, "_host", False)
  for a, b in zip(with_host, run()):
    assert torch.equal(a, b)


@pytest.mark.parametrize("sizes", [[1], [7, 2048, 5000], [3] * 500, [1 << 22, 12345], [5] * 3000])
@pytest.mark.parametrize("max_norm", [0.1, 1e9])
def test_clip_factor(sizes, max_norm):
  from t5x_b200.ops import native
  gen = torch.Generator(device="cuda").manual_seed(len(sizes))
  items, grads = native.AdamwItems(), []
  for n in sizes:
    g = torch.randn(n, device="cuda", generator=gen)
    grads.append(g)
    p, mu, nu = (torch.empty(n, device="cuda") for _ in range(3))
    items.add(p, g, mu, nu)
  got = native.grad_clip_scale(items, max_norm, "cuda")
  norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
  # eight products in 32 bits before the sum goes on in 64: a relative error of 8 * 2^-24, half of it in the root
  assert abs(float(got) / min(1.0, max_norm / norm) - 1) < 2 ** -20
  assert torch.equal(got, native.grad_clip_scale(items, max_norm, "cuda"))


def test_clip_of_no_gradients_and_of_values_that_are_not_finite():
  from t5x_b200.ops import native
  assert float(native.grad_clip_scale(native.AdamwItems(), 1.0, "cuda")) == 1.0
  for value, want in ((math.nan, math.nan), (math.inf, 0.0)):
    items = native.AdamwItems()
    g = torch.ones(3000, device="cuda")
    g[2999] = value
    t = [torch.zeros(3000, device="cuda") for _ in range(3)]
    items.add(t[0], g, t[1], t[2])
    got = float(native.grad_clip_scale(items, 1.0, "cuda"))
    assert got == want or (math.isnan(got) and math.isnan(want))


def test_values_that_are_not_finite_stay_in_their_block():
  p = {"w": torch.ones(1000, device="cuda")}
  opt = optimizers.adamw8(1e-2, weight_decay=0.0).create(p)
  g = torch.ones(1000, device="cuda")
  g[300] = math.nan
  opt = opt.apply_gradient({"w": g})
  bad = torch.isnan(p["w"])
  assert bad.nonzero().flatten().tolist() == [300]
  adam = adam_of(opt)
  assert torch.isnan(adam["mu_absmax"]["w"]).tolist() == [False, True, False, False]
  opt = opt.apply_gradient({"w": torch.ones(1000, device="cuda")})
  bad = torch.isnan(p["w"]).nonzero().flatten()
  assert bad.min() == 256 and bad.max() == 511


def test_zero_gradients_keep_zero_moments():
  p = {"w": torch.randn(700, device="cuda")}
  before = p["w"].clone()
  opt = optimizers.adamw8(1e-2, weight_decay=0.0).create(p)
  opt = opt.apply_gradient({"w": torch.zeros(700, device="cuda")})
  assert torch.equal(p["w"], before) and int(adam_of(opt)["nu"]["w"].sum()) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_that_stands_twice_is_stepped_in_turn(bits):
  """Two names of one tensor: the grouped launch would race, the parameters are stepped one after the other."""
  make = optimizers.adamw if bits == 32 else optimizers.adamw8
  g = {"a": torch.full((5000,), 0.5, device="cuda"), "b": torch.full((5000,), -1.0, device="cuda")}
  w = torch.linspace(-1, 1, 5000, device="cuda")
  want = w.cpu()
  make(1e-2, weight_decay=0.0).create({"a": w, "b": w}).apply_gradient(g)
  for x in (0.5, -1.0):  # a first step of Adam is lr * sign(g)
    want = want - 1e-2 * math.copysign(1, x)
  assert torch.allclose(w.cpu(), want, rtol=0, atol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_what_the_grouped_step_leaves_alone(bits):
  """Gradients of another type, weights that are not contiguous: the general path takes them and agrees."""
  make = optimizers.adamw if bits == 32 else optimizers.adamw8
  gen = torch.Generator(device="cuda").manual_seed(0)
  w, g = torch.randn(40, 30, device="cuda", generator=gen), torch.randn(40, 30, device="cuda", generator=gen)
  g = g.to(torch.bfloat16).float()
  plain = make(1e-2).create({"w": w.clone()}).apply_gradient({"w": g}).target["w"]
  half = make(1e-2).create({"w": w.clone()}).apply_gradient({"w": g.to(torch.bfloat16)}).target["w"]
  turned = make(1e-2).create({"w": w.clone().t()}).apply_gradient({"w": g.t()}).target["w"].t()
  for other in (half, turned):
    assert torch.allclose(other, plain, rtol=0, atol=1e-6)


def test_another_stream_and_a_captured_step():
  """On a stream of its own; captured once and replayed, with the step that it was captured with."""
  g = tree(SIZES, 7, bf16=False)
  make = lambda: optimizers.chain([optimizers.clip_by_global_norm(0.5), optimizers._adamw8(1e-2)])  # noqa: E731
  want = make().create(tree(SIZES, 1)).apply_gradient(g)
  got = make().create(tree(SIZES, 1))
  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    done = got.apply_gradient(g)
  torch.cuda.current_stream().wait_stream(stream)
  for a, b in zip(leaves(done.target), leaves(want.target)):
    assert torch.equal(a, b)
  replayed = make().create(tree(SIZES, 1))
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    replayed.apply_gradient(g)
  graph.replay()
  for a, b in zip(leaves(replayed.target), leaves(want.target)):
    assert torch.equal(a, b)


def test_draws_next_to_their_border():
  """First moments among the numbers whose steps are the same, each some 2^-22 of a step below the place from which
  its draw rounds it up: every code is that of the formula, whose sum of value and draw is exact in 64 bits."""
  n, seed = 64 * 256, 9
  up = ((optimizers._moment_noise(n, seed, 1, "cuda") & 0xFFFF).double() + 0.5) / 65536
  g = ((2 - up - 2.0 ** -22) * 2.0 ** -9 / 448).float()
  g[::256] = 1.0
  opt = optimizers.chain([optimizers._adamw8(1e-3, seed=seed)]).create({"a": {"w": torch.zeros(n, device="cuda")}})
  got = leaves(adam_of(opt.apply_gradient({"a": {"w": g}}))["mu"])[0]
  m = ((1 - 0.9) * g).view(-1, 256)
  y = m / m.amax(1, keepdim=True) * 448  # (rounded as before the draw)
  small = y < 2.0 ** -6
  want = torch.floor(y.double() * 2.0 ** 9 + up.view(-1, 256)) * 2.0 ** -9
  assert int(small.sum()) == 64 * 255 and float((want[small] == 2.0 ** -9).double().mean()) > 0.2
  assert torch.equal(got.view(torch.float8_e4m3fn).double().view(-1, 256)[small], want[small])
