"""Products in 8-bit integers of rows and channels far from 1: results that a type holds come out, whatever their factors are."""
import pytest
import torch

from t5x_b200.ops import functional as F
from t5x_b200.ops import native
from t5x_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


# one row, two, a few over a cluster (whole fours of channels and not), tiles of 256 (whole sectors of channels and not)
@pytest.mark.parametrize("rows,k,n", [(1, 300, 130), (2, 64, 40), (2, 20000, 33), (40, 257, 200), (40, 128, 131), (257, 96, 40),
                                      (2600, 160, 2048), (2304, 96, 2301)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("one", [False, True])
def test_rows_and_channels_of_any_size(rows, k, n, dtype, one):
  """one: a single row and a single channel are far out, among ordinary ones."""
  gen = torch.Generator("cuda").manual_seed(rows)
  randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
  far = 13 if dtype == torch.float16 else 110 if dtype == torch.bfloat16 else 135  # (in 32 bits below the normal numbers too)
  by_row = torch.randint(-far, min(far, 110) + 1, (rows, 1), generator=gen, device="cuda")
  by_channel = torch.randint(-110, 111, (1, n), generator=gen, device="cuda")
  if one:
    by_row[torch.arange(rows, device="cuda") != rows // 2] = 0
    by_channel[:, torch.arange(n, device="cuda") != n // 3] = 0
    by_row[rows // 2], by_channel[0, n // 3] = -far, 100
  x = torch.ldexp(randn(rows, k), by_row).to(dtype)
  weight = F.quantize_weight(torch.ldexp(randn(k, n), by_channel))
  info = torch.finfo(dtype)
  for residual in (None, torch.ldexp(randn(rows, n), by_row + by_channel).clamp(info.min / 4, info.max / 4).to(dtype)):
    before = native.launch_count()
    y = F.linear8(x, weight, residual)
    assert native.launch_count() > before
    plus = torch.zeros((), dtype=torch.float64) if residual is None else residual.double()
    product = ref.linear8(x.double(), weight.codes[:, :k], weight.absmax)
    want = product + plus.to("cuda")
    # eight roundings in 32 bits of the product, and the last one; results below the smallest normal number may be 0
    bound = (product.abs() + want.abs()) * 2.0 ** -21 * (1 + info.eps) + info.eps / 2 * want.abs() + 2 * info.smallest_normal
    # (what rounds beyond the largest is infinite)
    edge = info.max * (1 - info.eps)
    fits = want.abs() <= edge
    assert bool(((y.double() - want).abs() <= bound)[fits].all())
    assert bool((y.double() / want >= 1 - info.eps)[~fits].all())
