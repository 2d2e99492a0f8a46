"""The experts' products, 8-bit products and the gradients' norm where offsets
pass 32 bits. Whole numbers, exact throughout; checked at rows and columns near
the ends, where a wrapped offset would read or write elsewhere."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position


@pytest.fixture(autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)
  yield
  torch.cuda.empty_cache()


def _need(gib):
  free, _ = torch.cuda.mem_get_info()
  if free < gib * 2**30:
    pytest.skip(f"needs {gib} GiB")


def _order(offsets):
  return dense.ExpertOrder(None, None, torch.tensor(
      offsets, dtype=torch.int32, device="cuda"))


def _whole(shape, dtype):
  return torch.randint(-3, 4, shape, dtype=torch.int8, device="cuda").to(dtype)


def test_many_rows():
  """More than 2^32 bytes of rows, of results and of both gradients' operands."""
  _need(60)
  n, k, m = 2_100_007, 1032, 1040
  x, w = _whole((n, k), torch.bfloat16), _whole((2, k, m), torch.bfloat16)
  order = _order([0, n - 300, n - 2])
  y = dense.expert_matmul(x, w, order)
  for a, b, e in ((0, 50, 0), (n - 400, n - 300, 0), (n - 300, n - 2, 1)):
    assert torch.equal(y[a:b], (x[a:b].double() @ w[e].double()).bfloat16())
  assert not y[n - 2:].any()
  q = dense.quantize_weights(w)
  assert torch.equal(dense.matmul_8bit(x, q, order), y)
  del y
  dy = torch.zeros((n, m), dtype=torch.bfloat16, device="cuda")
  dy[n - 200:] = _whole((200, m), torch.bfloat16)
  dy[:64] = _whole((64, m), torch.bfloat16)
  dx, dw = dense.expert_matmul_grad(dy, x, w, order)
  assert torch.equal(dx[n - 200:n - 2], (
      dy[n - 200:n - 2].double() @ w[1].double().t()).bfloat16())
  assert not dx[64:n - 200].any() and not dx[n - 2:].any()
  assert torch.equal(dw[0], (x[:64].double().t() @ dy[:64].double()).bfloat16())
  assert torch.equal(dw[1], (x[n - 200:n - 2].double().t() @
                             dy[n - 200:n - 2].double()).bfloat16())


def test_large_weights():
  """More than 2^31 weights: the last experts' are found and written."""
  _need(60)
  e, k, m = 68, 4104, 8200
  w = torch.zeros((e, k, m), dtype=torch.bfloat16, device="cuda")
  for i in (0, e - 2, e - 1):
    w[i] = _whole((k, m), torch.bfloat16)
  x = _whole((60, k), torch.bfloat16)
  counts = [20] + [0] * (e - 3) + [20, 20]
  offsets = [0]
  for c in counts:
    offsets.append(offsets[-1] + c)
  order = _order(offsets)
  y = dense.expert_matmul(x, w, order)
  expected = torch.cat([(x[a:a + 20].double() @ w[i].double())
                        for a, i in ((0, 0), (20, e - 2), (40, e - 1))])
  assert torch.equal(y, expected.bfloat16())
  assert torch.equal(dense.matmul_8bit(x, dense.quantize_weights(w), order), y)
  dy = _whole((60, m), torch.bfloat16)
  _, dw = dense.expert_matmul_grad(dy, x, w, order, with_rows=False)
  for a, i in ((0, 0), (20, e - 2), (40, e - 1)):
    assert torch.equal(dw[i], (x[a:a + 20].double().t() @
                               dy[a:a + 20].double()).bfloat16())
  assert not dw[1:e - 2].any()


def test_norm_of_many_values():
  """A tensor of more than 2^32 values: it goes in pieces."""
  _need(24)
  n = 2**32 + 12_345
  g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
  at = torch.tensor([0, 2**31 - 1, 2**31, 2**32 - 1, 2**32, n - 1],
                    device="cuda")
  g[at] = 2.0
  norm, factor = dense.gradient_norm([g], max_norm=1.0)
  assert abs(float(norm) - 24**0.5) < 1e-6
  dense.clip_gradients([g], 24**0.5 / 2)
  assert (g[at] == 1).all() and int((g != 0).sum()) == 6
