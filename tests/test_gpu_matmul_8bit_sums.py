"""Sums of 8-bit products (lib/nn/dense.py matmul_8bit) are float32 whatever the
result's type, for every size of tile.

Values are their own codes: multiples of 1/8 up to 3/8 and some of 64, which a
block with its power of two holds exactly. Products are multiples of 2^-6, and
the magnitudes of a sum stay below 2^18 (see _base), so every partial sum is a
multiple of 2^-6 of at most 24 bits: exact in float32 in any order. Powers of two
of rows, of columns of blocks, and of blocks along the sum (with the inverse in
the weights) change no bit of a result. So results are expected bit for bit:
the sum in 64 bits, rounded once.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

TYPES = [torch.float32, torch.bfloat16, torch.float16]
B = 128


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _order(offsets):
  return dense.ExpertOrder(None, None, torch.tensor(
      offsets, dtype=torch.int32, device="cuda"))


def _base(shape, g):
  """Multiples of 1/8 up to 3/8, one in 20 a 64 of either sign, float32. A sum
  of 1000 such products has magnitudes below 2^18 unless 63 of its places have
  a 64 on both sides, where 2 or 3 are expected."""
  x = torch.randint(-3, 4, shape, device="cuda", generator=g).float() / 8
  sign = torch.randint(0, 2, shape, device="cuda", generator=g).float() * 2 - 1
  return torch.where(torch.rand(shape, device="cuda", generator=g) < 0.05,
                     64 * sign, x)


def _powers(n, lo, hi, g):
  return torch.exp2(torch.randint(lo, hi + 1, (n,), device="cuda",
                                  generator=g).float())


def _spread(p, n):
  return p.repeat_interleave(B)[:n]


def _run(offsets, rows, inner, outer, dtype, plain=False):
  g = torch.Generator(device="cuda").manual_seed(rows + inner + outer)
  experts = len(offsets) - 1
  x, w = _base((rows, inner), g), _base((experts, inner, outer), g)
  # float16 holds less: results stay below 2^16.
  half = dtype == torch.float16
  of_rows = _powers(rows, -6, -3, g) if half else _powers(rows, -30, 30, g)
  along = _powers(-(-inner // B), -2, 2, g) if half else _powers(
      -(-inner // B), -10, 10, g)
  across = _powers(-(-outer // B), -3, 0, g) if half else _powers(
      -(-outer // B), -20, 20, g)
  of_rows = of_rows[:, None]
  along, across = _spread(along, inner), _spread(across, outer)
  q = (x * of_rows * along).to(dtype)
  assert torch.equal(q.float(), x * of_rows * along)
  v = w / along[:, None] * across
  q[offsets[-1]:] = float("nan")
  if plain:
    y = dense.matmul_8bit(q, dense.quantize_weights(v[0]))
  else:
    y = dense.matmul_8bit(q, dense.quantize_weights(v), _order(offsets))
  for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
    exact = x[a:b].double() @ w[e].double()
    assert float((x[a:b].double().abs() @ w[e].double().abs()).max()
                 if b > a else 0.0) < 2**18
    exact = (exact * of_rows[a:b].double() * across.double()).to(dtype)
    assert torch.equal(y[a:b], exact)
  assert not y[offsets[-1]:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner", [40, 128, 650, 1000])
@pytest.mark.parametrize("offsets,rows,outer", [
    ([0, 1], 1, 7), ([0, 40], 40, 264), ([0, 0, 33, 100, 101], 105, 300),
    ([0, 20, 300, 300, 701], 703, 129)])
def test_few_rows(offsets, rows, inner, outer, dtype):
  """Tiles of 32 rows."""
  _run(offsets, rows, inner, outer, dtype)
  if len(offsets) == 2:
    _run(offsets, rows, inner, outer, dtype, plain=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner", [130, 650])
@pytest.mark.parametrize("offsets,rows,outer", [
    ([0, 3999], 3999, 1000), ([0, 1500, 1500, 1629, 3990], 4001, 1000)])
def test_more_rows(offsets, rows, inner, outer, dtype):
  """Tiles of 128 x 128: 256 of them, more than three quarters of the CUs."""
  _run(offsets, rows, inner, outer, dtype)
  if len(offsets) == 2:
    _run(offsets, rows, inner, outer, dtype, plain=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner", [130, 650])
@pytest.mark.parametrize("offsets,rows,outer", [
    ([0, 32_000], 32_000, 1000), ([0, 7000, 7000, 20_777, 31_990], 32_001,
                                  1000)])
def test_many_rows(offsets, rows, inner, outer, dtype):
  """Tiles of 256 x 256: 500 of them, two rounds of the CUs all but full."""
  _run(offsets, rows, inner, outer, dtype)
  if len(offsets) == 2:
    _run(offsets, rows, inner, outer, dtype, plain=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_small_products_beside_large_ones(dtype):
  """256 * 256 and its opposite leave the products of one."""
  x = torch.ones((70, 128), dtype=dtype, device="cuda")
  w = torch.ones((128, 9), dtype=dtype, device="cuda")
  x[:, 40:42] = 256
  w[40], w[41] = 256, -256
  y = dense.matmul_8bit(x, dense.quantize_weights(w))
  assert (y == 126).all()
