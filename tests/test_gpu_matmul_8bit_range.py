"""8-bit products (lib/nn/dense.py matmul_8bit) of blocks whose power of two is
near float32's ends, where a code times its power is past what 16 bits with
float32's exponents hold: 256 * 2^120, and codes below 2^-7 at 2^-126.

All values are their own codes but the largest float32, whose code is 256 (it is
256 * 2^120 less half an ulp), products are whole numbers times one power of two,
and their sums stay below 2^24 of it: exact in float32 in any order, expected bit
for bit.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

WIDE = [torch.float32, torch.bfloat16]
# Tiles of 32, 128 and 256 rows.
SIZES = [(50, 300, 140), (4000, 300, 1000), (32_000, 260, 1000)]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _whole(shape, seed, most=3):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return torch.randint(-most, most + 1, shape, device="cuda",
                       generator=g).double()


def _typed(x, dtype):
  # By way of float32: values below its normal ones stay.
  y = x.float()
  assert torch.equal(y.double(), x)
  return y.to(dtype)


def _check(y, exact, dtype):
  assert torch.equal(y, exact.float().to(dtype))


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_largest_values(rows, inner, outer, dtype):
  x, w = _whole((rows, inner), 1), _whole((inner, outer), 2)
  w[:, ::3] = 0  # nothing times the largest is nothing
  q = _typed(x * 2.0**120, dtype)
  # Some rows only, some of their blocks only.
  q[::3, 5], q[1::3, 200] = torch.finfo(dtype).max, -torch.finfo(dtype).max
  x[::3, 5], x[1::3, 200] = 256, -256
  small = _typed(w * 2.0**-100, torch.float32)
  y = dense.matmul_8bit(q, dense.quantize_weights(small))
  _check(y, x @ w * 2.0**20, dtype)
  # The weights' blocks, the other way about: three columns of blocks, one of
  # which has the largest.
  u = _typed(w * 2.0**120, torch.float32)
  u[7, 1] = torch.finfo(torch.float32).max
  w[7, 1] = 256
  x = _whole((rows, inner), 3)
  y = dense.matmul_8bit(_typed(x * 2.0**-100, dtype),
                        dense.quantize_weights(u))
  _check(y, x @ w * 2.0**20, dtype)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_smallest_values(rows, inner, outer, dtype):
  """Codes 2^-9 to 7 * 2^-9 of 2^-126, beside rows and blocks of other sizes.
  (bfloat16 has steps of 2^-133 there: multiples of four.)"""
  most = 7 if dtype == torch.float32 else 1
  step = 2.0**-135 if dtype == torch.float32 else 2.0**-133
  x, w = _whole((rows, inner), 1, most), _whole((inner, outer), 2)
  q = x * step
  q[::2] = x[::2] * 2.0**-20
  y = dense.matmul_8bit(_typed(q, dtype), dense.quantize_weights(
      _typed(w * 2.0**110, torch.float32)))
  _check(y, q @ w * 2.0**110, dtype)
  # The weights' blocks.
  w = _whole((inner, outer), 3, 7)
  x = _whole((rows, inner), 4)
  u = w * 2.0**-135
  u[128:256] = w[128:256] * 2.0**-130
  y = dense.matmul_8bit(_typed(x * 2.0**110, dtype), dense.quantize_weights(
      _typed(u, torch.float32)))
  _check(y, x @ u * 2.0**110, dtype)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_small_products(rows, inner, outer, dtype):
  """Products whose smallest codes are below float32's normal values."""
  x, w = _whole((rows, inner), 1), _whole((inner, outer), 2)
  x[:, 17], w[17, :] = 256, 256
  y = dense.matmul_8bit(_typed(x * 2.0**-66, dtype), dense.quantize_weights(
      _typed(w * 2.0**-66, torch.float32)))
  _check(y, x @ w * 2.0**-132, dtype)


@pytest.mark.parametrize("dtype", [*WIDE, torch.float16])
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_blocks_of_zeros(rows, inner, outer, dtype):
  x, w = _whole((rows, inner), 1), _whole((inner, outer), 2)
  x[::3, :128] = 0
  x[1::5] = 0
  w[128:256, :128] = 0
  y = dense.matmul_8bit(_typed(x, dtype),
                        dense.quantize_weights(_typed(w, dtype)))
  _check(y, x @ w, dtype)


def test_each_expert_has_its_own():
  """Experts of ordinary, large and small weights, rows to match."""
  offsets = [0, 3000, 9000, 9001, 16_000]
  x, w = _whole((16_007, 260), 1), _whole((4, 260, 1000), 2)
  of_experts = [0, 120, -132, -126]
  q = x.clone()
  for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
    q[a:b] *= 2.0**-of_experts[e] if e < 2 else 2.0**100
  u = torch.stack([w[e] * 2.0**of_experts[e] for e in range(4)])
  q[offsets[-1]:] = 0
  y = dense.matmul_8bit(
      _typed(q, torch.float32),
      dense.quantize_weights(_typed(u, torch.float32)),
      dense.ExpertOrder(None, None, torch.tensor(offsets, dtype=torch.int32,
                                                 device="cuda")))
  for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
    _check(y[a:b], q[a:b] @ u[e], torch.float32)
  assert not y[offsets[-1]:].any()
