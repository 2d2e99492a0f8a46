"""AdamW's hyperparameters on the GPU as tensors whose memory does not hold
their value (views that are negated when read, zeros that were never written),
of other types, and with tangents."""

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


def _value(x, dtype):
  return torch.tensor(x, dtype=dtype, device="cuda")


def _negated(x, dtype):
  return torch._neg_view(_value(-x, dtype))  # pylint: disable=protected-access


def _zero(dtype):
  return torch._efficientzerotensor((), dtype=dtype, device="cuda")  # pylint: disable=protected-access


def _update(learning_rate, grad_scale, step):
  g = torch.Generator(device="cuda").manual_seed(3)
  p, grad = (torch.randn(700, device="cuda", generator=g) for _ in range(2))
  state = dense.init_adamw_state([p])
  dense.adamw_update([p], [grad], state, learning_rate=learning_rate,
                     grad_scale=grad_scale, step=step)
  return p, state.m, state.v


def _same(got, expected):
  for a, b in zip(got, expected, strict=True):
    assert torch.equal(a, b)


F, I = torch.float32, torch.int64


def test_negated_views():
  expected = _update(_value(0.25, F), _value(0.5, F), _value(3, I))
  _same(_update(_negated(0.25, F), _value(0.5, F), _value(3, I)), expected)
  _same(_update(_value(0.25, F), _negated(0.5, F), _value(3, I)), expected)
  _same(_update(_value(0.25, F), _value(0.5, F), _negated(3, I)), expected)


def test_zeros_that_were_never_written():
  _same(_update(_zero(F), _value(0.5, F), _value(3, I)),
        _update(_value(0.0, F), _value(0.5, F), _value(3, I)))
  _same(_update(_value(0.25, F), _zero(F), _value(3, I)),
        _update(_value(0.25, F), _value(0.0, F), _value(3, I)))


def test_other_types_and_shapes():
  expected = _update(_value(0.25, F), _value(0.5, F), _value(3, I))
  _same(_update(_value(0.25, torch.float64), _value([[0.5]], torch.bfloat16),
                _value([3], torch.int32)), expected)


def test_tangents_are_refused():
  with forward_ad.dual_level():
    x = _value(0.25, F)
    dual = forward_ad.make_dual(x, torch.ones_like(x))
    with pytest.raises(ValueError, match="tangent"):
      _update(dual, None, 1)
    with pytest.raises(ValueError, match="tangent"):
      _update(0.1, dual, 1)
