"""Forward-mode differentiation: the dense operators have none, and say so
instead of returning results without a tangent."""

import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad  # pylint: disable=g-import-not-at-top,wrong-import-position

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _calls():
  """name -> (operator of one tensor, that tensor)."""
  g = torch.Generator(device="cuda").manual_seed(0)
  new = lambda *s: torch.randn(s, device="cuda", generator=g)
  x, rows, w, gates = new(6, 8), new(12, 8), new(8), new(6, 2)
  order = dense.sort_by_expert(
      torch.randint(0, 3, (6, 2), device="cuda", generator=g), 3)
  _, mean, rstd = dense.layer_norm(x, w, return_stats=True)
  state = dense.init_adamw_state([w])
  update = lambda p, q: dense.adamw_update([p], [q], state, learning_rate=0.1)
  return {
      "norm": (lambda t: dense.layer_norm(t, w), x),
      "norm_weight": (lambda t: dense.layer_norm(x, t), w),
      "norm_bias": (lambda t: dense.layer_norm(x, None, t), w),
      "norm_grad": (lambda t: dense.layer_norm_grad(t, x, mean, rstd), x),
      "norm_grad_mean": (lambda t: dense.layer_norm_grad(x, x, t, rstd), mean),
      "to": (lambda t: dense.tokens_to_experts(t, order), x),
      "to_grad": (lambda t: dense.tokens_to_experts_grad(t, order), rows),
      "from": (lambda t: dense.tokens_from_experts(t, gates, order), rows),
      "from_weights": (lambda t: dense.tokens_from_experts(rows, t, order),
                       gates),
      "from_grad": (lambda t: dense.tokens_from_experts_grad(
          t, rows, gates, order), x),
      "adamw_param": (lambda t: update(t, x[0]), w),
      "adamw_grad": (lambda t: update(w, t), x[0]),
  }


NAMES = ["norm", "norm_weight", "norm_bias", "norm_grad", "norm_grad_mean",
         "to", "to_grad", "from", "from_weights", "from_grad", "adamw_param",
         "adamw_grad"]


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused(name):
  calls = _calls()
  assert list(calls) == NAMES
  f, t = calls[name]
  f(t)
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(t, torch.ones_like(t))
    with pytest.raises(ValueError, match="tangent"):
      f(dual)
    f(t)
  f(t)


@pytest.mark.parametrize("name", ["norm", "to", "from", "from_weights"])
def test_a_tangent_of_what_autograd_records_is_refused(name):
  f, t = _calls()[name]
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(t.clone().requires_grad_(), torch.ones_like(t))
    with pytest.raises((RuntimeError, ValueError)):
      f(dual)
