"""The experts' products of some of an order's experts (lib/nn/dense.py): the rows
before the first one's are rows of none, as those behind the last one's are. They
are not read and give zeros."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _whole(shape, dtype, seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return torch.randint(-3, 4, shape, device="cuda", generator=g).to(dtype)


def _after(call, *likes):
  """call()'s results; memory that the allocator hands out next holds NaN."""
  for like in likes:
    stale = torch.full_like(like, float("nan"))
    del stale
  return call()


# Rows, the offsets of the experts taken, inner, outer: tiles of 32 rows, cut along
# the sum, 128 x 128 through registers, and 256 x 256.
CASES = [(60, [7, 7, 30, 50], 40, 24), (60, [59, 60], 40, 24),
         (60, [60, 60], 40, 24), (90, [33, 64, 90], 4096, 40),
         (30_001, [9001, 9001, 20_000, 29_000], 100, 131),
         (32_000, [300, 12_345, 31_000], 264, 1000),
         (300, [5 + 2 * i for i in range(130)], 40, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,offsets,inner,outer", CASES)
def test_rows_before_the_first(n, offsets, inner, outer, dtype):
  experts, a, b = len(offsets) - 1, offsets[0], offsets[-1]
  x, dy = _whole((n, inner), dtype, 1), _whole((n, outer), dtype, 2)
  w = _whole((experts, inner, outer), dtype, 3)
  order = dense.ExpertOrder(None, None, torch.tensor(
      offsets, dtype=torch.int32, device="cuda"))
  # The same experts after one that has the rows before.
  all_order = dense.ExpertOrder(None, None, torch.tensor(
      [0] + offsets, dtype=torch.int32, device="cuda"))
  all_w = torch.cat([torch.zeros_like(w[:1]), w])
  y = dense.expert_matmul(x, all_w, all_order)
  dx, dw = dense.expert_matmul_grad(dy, x, all_w, all_order)
  y8 = dense.matmul_8bit(x, dense.quantize_weights(all_w), all_order)
  x[:a], dy[:a] = float("nan"), float("inf")
  x[b:], dy[b:] = float("nan"), float("inf")
  assert torch.equal(_after(lambda: dense.expert_matmul(x, w, order), y, y), y)
  got = _after(lambda: dense.expert_matmul_grad(dy, x, w, order), dw, dx)
  assert torch.equal(got[0], dx) and torch.equal(got[1], dw[1:])
  q = dense.quantize_weights(w)
  assert torch.equal(_after(lambda: dense.matmul_8bit(x, q, order), y8, y8), y8)
