"""The gradients' norm and clipping (lib/nn/dense.py) follow no graph: gradients
that autograd would follow are refused, not taken for constants."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _grads(create_graph, stride=1):
  x = torch.arange(1.0, 41.0, device="cuda").requires_grad_()
  g, = torch.autograd.grad((x**3).sum(), x, create_graph=create_graph)
  return [torch.ones(5, device="cuda"), None, g[::stride]]


@pytest.mark.parametrize("stride", [1, 2])
def test_gradients_with_a_graph(stride):
  grads = _grads(True, stride)
  before = grads[2].detach().clone()
  for call in (lambda: dense.gradient_norm(grads),
               lambda: dense.gradient_norm(grads, max_norm=1.0),
               lambda: dense.clip_gradients(grads, 1.0)):
    with pytest.raises(ValueError, match=r"grads\[2\]"):
      call()
  assert torch.equal(grads[2].detach(), before)
  assert (grads[0] == 1).all()


def test_without_a_graph():
  grads, same = _grads(True), _grads(False)
  expected = dense.gradient_norm(same)
  with torch.no_grad():
    assert torch.equal(dense.gradient_norm(grads), expected)
  detached = [g if g is None else g.detach() for g in grads]
  assert torch.equal(dense.gradient_norm(detached), expected)
  assert torch.equal(dense.clip_gradients(same, 1.0), expected)
  # A weight's own .grad, as a backward pass leaves it.
  w = torch.ones(7, device="cuda").requires_grad_()
  (2 * w).sum().backward()
  assert abs(float(dense.gradient_norm([w.grad])) - 28**0.5) < 1e-6
  dense.clip_gradients([w.grad], 0.5)
