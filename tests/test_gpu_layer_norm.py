"""Layer norm and its gradients (lib/nn/dense.py) against the definition in
64 bits, at the widths where the kernels change layout, with odd strides,
missing weights, and rows that are constant or not finite.

Tolerances. u is float32's unit roundoff, uo the result's. A lane adds at most
40 values, then come at most 6 steps over lanes and 16 wavefronts: a sum of n
values is off by at most 64 u times the sum of magnitudes. So the mean is off
by 64 u max|x|, a deviation by that and its own rounding, the variance by 64 u
of itself (an error of the mean enters it squared), and
  |y - exact| <= uo |y| + 256 u max|x| rstd |w| + 2 u |b|.
The gradients are held the same way, by sums of magnitudes. Halves below the
smallest normal number have an absolute rounding instead (2^-25).
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

U = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8,
         torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _inputs(rows, dim, dtype, seed=0, shift=1.0):
  g = torch.Generator(device="cuda").manual_seed(seed)
  x = torch.randn((rows, dim), device="cuda", generator=g)
  x = x * torch.rand((rows, 1), device="cuda", generator=g) + shift
  w = 1 + 0.2 * torch.randn(dim, device="cuda", generator=g)
  b = 0.2 * torch.randn(dim, device="cuda", generator=g)
  dy = torch.randn((rows, dim), device="cuda", generator=g)
  return x.to(dtype), w, b, dy.to(dtype)


def _exact(x, w, b, eps=EPS):
  x = x.double()
  mean = x.mean(-1, keepdim=True)
  rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
  y = (x - mean) * rstd
  if w is not None:
    y = y * w.double()
  if b is not None:
    y = y + b.double()
  return y, mean, rstd


def _check_forward(x, w, b, y):
  exact, _, rstd = _exact(x, w, b)
  top = x.double().abs().amax(-1, keepdim=True)
  wm = 1.0 if w is None else w.double().abs()
  bm = 0.0 if b is None else b.double().abs()
  tol = (ROUND[y.dtype] * exact.abs() + 256 * U * top * rstd * wm + 2 * U * bm +
         TINY[y.dtype])
  assert y.dtype == x.dtype and y.shape == x.shape
  assert ((y.double() - exact).abs() <= tol).all()


def _check_backward(x, w, dy, mean, rstd, got):
  dx, dw, db = got
  mean, rstd = mean.double().reshape(-1, 1), rstd.double().reshape(-1, 1)
  xd, dyd = x.double(), dy.double()
  xhat = (xd - mean) * rstd
  h = dyd if w is None else dyd * w.double()
  exact = rstd * (h - h.mean(1, keepdim=True) -
                  xhat * (h * xhat).mean(1, keepdim=True))
  # xhat in float32: two roundings of x - mean and of the product.
  xerr = 4 * U * (xd.abs() + mean.abs()) * rstd
  along = (h * xhat).abs().mean(1, keepdim=True)
  tol = ROUND[dx.dtype] * exact.abs() + TINY[dx.dtype] + rstd * (
      128 * U * (h.abs() + h.abs().mean(1, keepdim=True) + xhat.abs() * along) +
      xerr * along + xhat.abs() * (h.abs() * xerr).mean(1, keepdim=True))
  assert dx.dtype == x.dtype
  assert ((dx.double() - exact).abs() <= tol).all()
  if dw is not None:
    exact = (dyd * xhat).sum(0)
    tol = (ROUND[dw.dtype] * exact.abs() + TINY[dw.dtype] +
           256 * U * (dyd * xhat).abs().sum(0) + (dyd.abs() * xerr).sum(0))
    assert ((dw.double() - exact).abs() <= tol).all()
  if db is not None:
    exact = dyd.sum(0)
    tol = (ROUND[db.dtype] * exact.abs() + TINY[db.dtype] +
           256 * U * dyd.abs().sum(0))
    assert ((db.double() - exact).abs() <= tol).all()


DIMS = [1, 2, 3, 7, 8, 16, 17, 32, 64, 65, 100, 128, 129, 255, 256, 260, 512,
        513, 1000, 1024, 1025, 2048, 2056, 3328, 4096, 4104, 8192, 8193, 16384,
        16392, 20001, 32768, 40000]


@pytest.mark.parametrize("dtype", list(ROUND), ids=str)
@pytest.mark.parametrize("dim", DIMS)
def test_forward_and_backward(dim, dtype):
  print("dim", dim, dtype, flush=True)
  rows = 37 if dim <= 4096 else 5
  for wtype in {torch.float32, dtype}:
    x, w, b, dy = _inputs(rows, dim, dtype, seed=dim)
    w, b = w.to(wtype), b.to(wtype)
    y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
    _check_forward(x, w, b, y)
    assert torch.equal(y, dense.layer_norm(x, w, b, epsilon=EPS))
    got = dense.layer_norm_grad(dy, x, mean, rstd, w)
    assert got[1].dtype == wtype and got[2].dtype == wtype
    _check_backward(x, w, dy, mean, rstd, got)
    again = dense.layer_norm_grad(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("rows", [0, 1, 2, 3, 64, 1023, 4099])
@pytest.mark.parametrize("dim", [12, 100, 520, 1032])
def test_numbers_of_rows(rows, dim):
  x, w, b, dy = _inputs(rows, dim, torch.bfloat16, seed=rows)
  y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  _check_forward(x, w, b, y)
  got = dense.layer_norm_grad(dy, x, mean, rstd, w)
  _check_backward(x, w, dy, mean, rstd, got)
  if rows == 0:
    assert (got[1] == 0).all() and (got[2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("weighted", [(0, 0), (1, 0), (0, 1)])
def test_missing_weight_or_bias(weighted, dtype):
  x, w, b, dy = _inputs(50, 96, dtype)
  w = w if weighted[0] else None
  b = b if weighted[1] else None
  y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  _check_forward(x, w, b, y)
  got = dense.layer_norm_grad(dy, x, mean, rstd, w, with_bias=b is not None)
  assert (got[1] is None) == (w is None) and (got[2] is None) == (b is None)
  _check_backward(x, w, dy, mean, rstd, got)


@pytest.mark.parametrize("dim", [24, 100, 1024])
def test_strides(dim):
  """Rows inside a wider matrix (aligned and not), a transposed matrix, one
  row repeated, and more dimensions."""
  g = torch.Generator(device="cuda").manual_seed(1)
  wide = torch.randn((40, dim + 24), device="cuda", generator=g)
  _, w, b, _ = _inputs(1, dim, torch.float32)
  views = [wide[:, 8:8 + dim], wide[:, 3:3 + dim], wide[::3, :dim],
           torch.randn((dim, 40), device="cuda", generator=g).t(),
           wide[5:6, :dim].expand(40, dim)]
  for x in views:
    y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
    _check_forward(x, w, b, y)
    for dy in (wide[:x.shape[0], 1:1 + dim],
               torch.ones((1, 1), device="cuda").expand(x.shape)):
      got = dense.layer_norm_grad(dy, x, mean, rstd, w)
      _check_backward(x, w, dy, mean, rstd, got)
  x = wide[:, :dim].reshape(4, 5, 2, dim)
  y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  assert y.shape == x.shape and mean.shape == rstd.shape == (4, 5, 2)
  _check_forward(x, w, b, y)
  _check_forward(x[0, 0, 0], w, b,
                 dense.layer_norm(x[0, 0, 0], w, b, epsilon=EPS))
  weights = torch.randn((dim, 2), device="cuda", generator=g)
  _check_forward(x, weights[:, 0], weights[:, 1],
                 dense.layer_norm(x, weights[:, 0], weights[:, 1],
                                  epsilon=EPS))
  shifted = torch.randn(dim + 1, device="cuda", generator=g)[1:]
  _check_forward(x, shifted, b, dense.layer_norm(x, shifted, b, epsilon=EPS))


def test_large_mean_keeps_the_deviation():
  x, w, b, _ = _inputs(64, 1024, torch.float32, shift=1000.0)
  _check_forward(x, w, b, dense.layer_norm(x, w, b, epsilon=EPS))


def test_constant_and_not_finite_rows():
  x, w, b, dy = _inputs(8, 200, torch.float32)
  x[1] = 0.25
  x[3, 7] = float("inf")
  x[5, 0] = float("nan")
  x[6] = 0.0
  y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  fine = torch.tensor([0, 1, 2, 4, 6, 7], device="cuda")
  _check_forward(x[fine], w, b, y[fine])
  assert torch.equal(y[6], b) and torch.equal(y[1], b)
  assert y[3].isnan().all() and y[5].isnan().all()
  got = dense.layer_norm_grad(dy, x, mean, rstd, w)
  assert got[0][fine].isfinite().all() and got[1].isnan().all()
  assert got[0][3].isnan().all() and got[0][5].isnan().all()
  assert got[2].isfinite().all()


def test_autograd_and_differences():
  x, w, b, c = _inputs(9, 40, torch.float32, seed=4)
  p = [v.clone().requires_grad_() for v in (x, w, b)]
  (dense.layer_norm(*p, epsilon=EPS) * c).sum().backward()
  _, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  direct = dense.layer_norm_grad(c, x, mean, rstd, w)
  for q, d in zip(p, direct):
    assert torch.equal(q.grad, d)
  g = torch.Generator(device="cuda").manual_seed(9)
  f = lambda *v: (_exact(*v)[0] * c.double()).sum()
  args = [v.double() for v in (x, w, b)]
  for i, grad in enumerate(direct):
    d = torch.randn(args[i].shape, device="cuda", generator=g).double()
    h = 1e-5
    up = [a + h * d if j == i else a for j, a in enumerate(args)]
    down = [a - h * d if j == i else a for j, a in enumerate(args)]
    slope = (f(*up) - f(*down)) / (2 * h)
    along = (grad.double() * d)
    # Differences are off by h^2 of the third derivative (rows here have
    # rstd < 200) and by 1e-16 / h; gradients by float32's rounding.
    assert (along.sum() - slope).abs() <= 1e-5 * along.abs().sum() + 1e-4


def test_autograd_of_parts():
  """Gradients that nobody asks for are not returned; broadcast gradients."""
  x, w, b, _ = _inputs(6, 32, torch.bfloat16)
  w = w.requires_grad_()
  y, mean, _ = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  assert not mean.requires_grad
  y.sum().backward()
  assert w.grad is not None and x.grad is None
  x = x.requires_grad_()
  dense.layer_norm(x.view(2, 3, 32)).float().mean().backward()
  assert x.grad.shape == x.shape


def test_other_stream():
  x, w, b, _ = _inputs(512, 768, torch.float32)
  expected = dense.layer_norm(x, w, b)
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    got = dense.layer_norm(x * 1.0, w, b)
  torch.cuda.current_stream().wait_stream(s)
  assert torch.equal(got, expected)


def test_many_rows_and_offsets_past_32_bits():
  """Element offsets above 2^31 (a view of rows far apart)."""
  rows, dim, stride = 5, 64, 1 << 29
  big = torch.empty((rows - 1) * stride + dim, dtype=torch.bfloat16,
                    device="cuda")
  x = big.as_strided((rows, dim), (stride, 1))
  values, w, b, dy = _inputs(rows, dim, torch.bfloat16)
  x.copy_(values)
  y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  _check_forward(values, w, b, y)
  got = dense.layer_norm_grad(dy, x, mean, rstd, w)
  _check_backward(values, w, dy, mean, rstd, got)


@pytest.mark.parametrize("dim", [1024, 1001])
def test_more_than_the_caches(dim):
  """Calls of more than 256 MB read their rows past the caches: the same bits
  as calls on parts of the rows, and sums over all of them."""
  rows = 50000
  x, w, b, dy = _inputs(rows, dim, torch.bfloat16)
  y, mean, rstd = dense.layer_norm(x, w, b, epsilon=EPS, return_stats=True)
  dx, dw, db = dense.layer_norm_grad(dy, x, mean, rstd, w)
  sums = torch.zeros((2, dim), dtype=torch.float64, device="cuda")
  size = torch.zeros((2, dim), dtype=torch.float64, device="cuda")
  for at in range(0, rows, 10000):
    cut = slice(at, at + 10000)
    part = dense.layer_norm(x[cut], w, b, epsilon=EPS)
    assert torch.equal(part, y[cut])
    part = dense.layer_norm_grad(dy[cut], x[cut], mean[cut], rstd[cut], w)
    assert torch.equal(part[0], dx[cut])
    xhat = (x[cut].double() - mean[cut, None].double()) * rstd[cut, None].double()
    for i, v in enumerate((dy[cut].double() * xhat, dy[cut].double())):
      sums[i] += v.sum(0)
      size[i] += v.abs().sum(0)
  # A lane adds a row at a time, 3 work-groups of 4 rows a CU: 17 rows of it,
  # then 4 and 768 / 32 sums; and xhat is off by 4 u (|x| + |mean|) rstd < 32 u.
  assert ((dw - sums[0]).abs() <= 64 * U * size[0] + 32 * U * size[1]).all()
  assert ((db - sums[1]).abs() <= 64 * U * size[1]).all()


def test_refusals():
  x, w, b, dy = _inputs(4, 16, torch.bfloat16)
  y, mean, rstd = dense.layer_norm(x, w, b, return_stats=True)
  bad = [
      lambda: dense.layer_norm(x.cpu(), w, b),
      lambda: dense.layer_norm(x.double(), w, b),
      lambda: dense.layer_norm(x.tolist()),
      lambda: dense.layer_norm(x, w[:8], b),
      lambda: dense.layer_norm(x, w, b.bfloat16()),
      lambda: dense.layer_norm(x, w.half(), b.half()),
      lambda: dense.layer_norm(x, w, b, epsilon=-1.0),
      lambda: dense.layer_norm(x[0, 0]),
      lambda: dense.layer_norm(x[:, :0]),
      lambda: dense.layer_norm_grad(dy[:3], x, mean, rstd, w),
      lambda: dense.layer_norm_grad(dy.float(), x, mean, rstd, w),
      lambda: dense.layer_norm_grad(dy, x, mean[:3], rstd, w),
      lambda: dense.layer_norm_grad(dy, x, mean, rstd.double(), w),
  ]
  for call in bad:
    with pytest.raises(ValueError):
      call()
  assert y.isfinite().all()
