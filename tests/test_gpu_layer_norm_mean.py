"""Layer norm of rows whose mean is large against their deviations: constant
rows and nearly constant ones, where the first mean's rounding is as large as
what is left of the row.

Tolerances. u is float32's unit roundoff, and a sum of n values is off by at
most 64 u times the sum of magnitudes (a lane's values, the lanes, the
wavefronts). The first mean is then off by c <= 64 u max|x|, plus u of itself,
and what is left of the row has the mean c, the mean square s^2 + c^2 (s: the
row's deviation) and a mean magnitude of at most s + c. So the shift is off by
66 u (s + c), a deviation by that and 2 u of its own magnitude d <= |x - mean| +
c, and the variance by 66 u (s^2 + c^2) + 2 c * 66 u (s + c) + 2 u c^2, which is
below 512 u (s^2 + c^2). With that
  |mean off|  <= u |mean| + 66 u (s + c),
  |rstd off|  <= rstd (256 u (s^2 + c^2) rstd^2 + 4 u),
  |xhat off|  <= rstd (66 u (s + c) + 4 u d)
                 + |xhat| (256 u (s^2 + c^2) rstd^2 + 4 u),
where the terms in (s^2 + c^2) rstd^2 are first-order (they stay below 0.1).
Nothing here grows with max|x| * rstd: c enters times u.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

U = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8,
         torch.float16: 2.0**-11}
# Halves below the smallest normal number have an absolute rounding.
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _check(x, w, b, y, mean, rstd):
  xd, wd, bd = x.double(), w.double(), b.double()
  mu = xd.mean(1, keepdim=True)
  s2 = (xd - mu).square().mean(1, keepdim=True)
  s, r = s2.sqrt(), (s2 + EPS).rsqrt()
  xhat = (xd - mu) * r
  exact = xhat * wd + bd
  c = 66 * U * xd.abs().amax(1, keepdim=True)
  part = 256 * U * (s2 + c * c) * r * r + 4 * U
  assert (part < 0.1).all()
  d = (xd - mu).abs() + c
  off = r * (66 * U * (s + c) + 4 * U * d) + xhat.abs() * part
  tol = ROUND[y.dtype] * exact.abs() + 1.01 * off * wd.abs() + 2 * U * (
      bd.abs() + exact.abs()) + TINY[y.dtype]
  assert ((y.double() - exact).abs() <= tol).all()
  tol = U * mu.abs() + 66 * U * (s + c)
  assert ((mean.double().unsqueeze(1) - mu).abs() <= tol).all()
  assert ((rstd.double().unsqueeze(1) - r).abs() <= 1.01 * part * r).all()


DIMS = [3, 7, 65, 100, 200, 1000, 1024, 1025, 3331, 4100, 8200, 16390, 20001]
# Values of a row that are no short binary fractions.
CONSTANT = [0.1, -777.7, 1000.3, 10000.3]


@pytest.mark.parametrize("dtype", list(ROUND), ids=str)
@pytest.mark.parametrize("dim", DIMS)
def test_constant_rows(dim, dtype):
  print("dim", dim, dtype, flush=True)
  x = torch.tensor(CONSTANT, device="cuda").unsqueeze(1).expand(-1, dim)
  x = x.to(dtype)
  g = torch.Generator(device="cuda").manual_seed(dim)
  w = 1 + 0.2 * torch.randn(dim, device="cuda", generator=g)
  b = 0.2 * torch.randn(dim, device="cuda", generator=g)
  y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  assert torch.equal(y, dense.layer_norm(x, w, b, epsilon=EPS))
  _check(x, w, b, y, mean, rstd)


@pytest.mark.parametrize("deviation", [1e-3, 0.03])
@pytest.mark.parametrize("dim", DIMS)
def test_nearly_constant_rows(dim, deviation):
  print("dim", dim, deviation, flush=True)
  g = torch.Generator(device="cuda").manual_seed(dim)
  values = torch.tensor(CONSTANT[1:], device="cuda").unsqueeze(1)
  x = values + deviation * torch.randn((3, dim), device="cuda", generator=g)
  w = 1 + 0.2 * torch.randn(dim, device="cuda", generator=g)
  b = 0.2 * torch.randn(dim, device="cuda", generator=g)
  y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  assert torch.equal(y, dense.layer_norm(x, w, b, epsilon=EPS))
  _check(x, w, b, y, mean, rstd)


def test_squares_past_float32():
  """Deviations whose squares overflow: the reciprocal deviation is zero and
  the result the bias, no NaN of infinity minus infinity."""
  x = torch.tensor([[1.0, -1.0, 0.3, 0.7, 5.0]], device="cuda") * 1e30
  b = torch.arange(5.0, device="cuda")
  y, _, rstd = dense.layer_norm(x, None, b, return_stats=True)
  assert (rstd == 0).all() and torch.equal(y[0], b)
