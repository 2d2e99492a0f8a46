"""AdamW's count of steps where it changes between a value on the GPU and the
host: the bias corrections never start again by themselves."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

RATE = 0.01


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _run(bits, updates, resume):
  """Three steps counted on the GPU, then what `resume` does for the fourth."""
  g = torch.Generator(device="cuda").manual_seed(1)
  p = torch.randn(300, device="cuda", generator=g)
  grads = [torch.randn(300, device="cuda", generator=g) for _ in range(5)]
  state = dense.init_adamw_state([p], state_bits=bits)
  count = torch.zeros((), dtype=torch.int64, device="cuda")
  for i in range(3):
    count += 1
    updates([p], [grads[i]], state, count)
  state = resume(p, grads[3], state, count)
  if state is not None:
    dense.adamw_update([p], [grads[4]], state, learning_rate=RATE)
    assert state.step == 5
  return p


def _on_gpu(p, g, state, count):
  dense.adamw_update(p, g, state, learning_rate=RATE, step=count)


def _on_host(p, g, state, _):
  dense.adamw_update(p, g, state, learning_rate=RATE)


def _next(p, g, state, _):
  dense.adamw_update([p], [g], state, learning_rate=RATE)
  return state


def _explicit(p, g, state, count):
  with pytest.raises(ValueError, match="counted on the GPU"):
    dense.adamw_update([p], [g], state, learning_rate=RATE)
  dense.adamw_update([p], [g], state, learning_rate=RATE, step=int(count) + 1)
  return state


def _set(p, g, state, count):
  state.step = int(count)
  return _next(p, g, state, count)


def _restored(p, g, state, count):
  """A checkpoint as the class describes it."""
  new = dense.init_adamw_state([p], state_bits=state.bits)
  for name in ("m", "v", "m_scale", "v_scale"):
    if getattr(state, name) is not None:
      getattr(new, name).copy_(getattr(state, name))
  new.step = int(count)
  return _next(p, g, new, count)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("resume", [_explicit, _set, _restored],
                         ids=lambda f: f.__name__)
def test_from_the_gpu_to_the_host(bits, resume):
  expected = _run(bits, _on_host, _next)
  got = _run(bits, _on_gpu, resume)
  # Factors are made in 64 bits on either side and may differ in float32's last
  # bit, and so may each of the steps' few products: the weights are of order 1
  # and a step moves them by about RATE.
  assert ((got - expected).abs() <= 2.0**-20 * (expected.abs() + RATE)).all()


def test_a_refused_step_changes_nothing():
  p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
  state = dense.init_adamw_state([p])
  count = torch.ones((), dtype=torch.int64, device="cuda")
  dense.adamw_update([p], [g], state, learning_rate=RATE, step=count)
  before, m = p.clone(), state.m.clone()
  with pytest.raises(ValueError):
    dense.adamw_update([p], [g], state, learning_rate=RATE)
  assert torch.equal(p, before) and torch.equal(state.m, m)
  count += 1
  dense.adamw_update([p], [g], state, learning_rate=RATE, step=count)
  assert not torch.equal(p, before)
