"""The gradients' norm and clipping (lib/nn/dense.py) against sums in 64 bits.

Squares of float32 values are exact in 64 bits, and a sum of n of them is off by
at most n 2^-53 of itself: nothing beside the norm's rounding to float32, half a
step (2^-24), which the tolerance of one step covers together with the factor's
quotient. A scaled value is one product (2^-24 and the factor's own step), rounded
once to its type.
"""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

STEP = 2.0**-23
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _tensors(sizes, types, seed=0, scale=1.0):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return [(scale * torch.randn(n, device="cuda", generator=g)).to(
      types[i % len(types)]) for i, n in enumerate(sizes)]


def _norm(tensors):
  return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


def _near(got, expected, steps=1):
  assert got.dtype == torch.float32 and got.shape == ()
  assert abs(float(got) - expected) <= steps * STEP * expected


SIZES = {
    "one": [1],
    "few": [1, 2, 3, 7, 8, 9, 63, 64, 65],
    "round": [4095, 4096, 4097, 8192, 0, 12289],
    "many": [1 + (i * 37) % 500 for i in range(400)],
    "large": [5_000_003, 40_000_000, 17],
    "whole": [1024] * 168,
    "one_more": [1024] * 169,
}


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("types", [[t] for t in TYPES] + [TYPES])
def test_norm(sizes, types):
  tensors = _tensors(SIZES[sizes], types)
  exact = _norm(tensors)
  _near(dense.gradient_norm(tensors), exact)
  for limit in (exact / 3, exact * 3, 0.0, math.inf):
    norm, factor = dense.gradient_norm(tensors, max_norm=limit)
    _near(norm, exact)
    _near(factor, min(1.0, limit / exact))


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_clip(sizes, dtype):
  tensors = _tensors(SIZES[sizes], [dtype])
  before = [t.clone() for t in tensors]
  exact = _norm(tensors)
  _near(dense.clip_gradients(tensors, 2 * exact), exact)
  for t, b in zip(tensors, before):
    assert torch.equal(t, b)
  limit = exact / 7
  _near(dense.clip_gradients(tensors, limit), exact)
  for t, b in zip(tensors, before):
    expected = b.double() * (limit / exact)
    # float16 has values below its smallest normal one, 2^-24 apart.
    bound = expected.abs() * (2 * STEP + torch.finfo(dtype).eps / 2)
    if dtype == torch.float16:
      bound = bound.clamp_min(2.0**-25 * 1.01)
    assert ((t.double() - expected).abs() <= bound).all()


def test_squares_past_float32():
  for scale in (1e30, 1e-30):
    tensors = _tensors([1000, 5], [torch.float32], scale=scale)
    exact = _norm(tensors)
    norm, factor = dense.gradient_norm(tensors, max_norm=exact / 10)
    _near(norm, exact)
    _near(factor, 0.1, 2)
  # The norm itself is past float32: infinite, and the factor is not.
  t = torch.full((100,), 3e38, device="cuda")
  norm, factor = dense.gradient_norm([t], max_norm=3e38)
  assert float(norm) == math.inf
  _near(factor, 0.1, 2)
  small = torch.full((3,), 1e-42, device="cuda")
  assert abs(float(dense.gradient_norm([small])) /
             _norm([small]) - 1) < 2.0**-9  # a subnormal of ten bits


def test_zeros_and_nothing():
  z = torch.zeros(10, device="cuda")
  for grads in ([], (), [None], [z], [z[:0]], [None, z, None]):
    norm, factor = dense.gradient_norm(grads, max_norm=1.0)
    assert float(norm) == 0 and float(factor) == 1
    assert float(dense.clip_gradients(grads, 1.0)) == 0
  assert not z.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(dtype):
  a, b = _tensors([5000, 300], [dtype])
  a[4999] = math.inf
  norm, factor = dense.gradient_norm([a, b], max_norm=1.0)
  assert float(norm) == math.inf and float(factor) == 0
  dense.clip_gradients([a, b], 1.0)
  assert not b.any() and not a[:4999].any() and a[4999].isnan()
  a, b = _tensors([5000, 300], [dtype])
  b[0] = math.nan
  norm, factor = dense.gradient_norm([a, b], max_norm=1.0)
  assert math.isnan(norm) and math.isnan(factor)
  dense.clip_gradients([a, b], 1.0)
  assert a.isnan().all() and b.isnan().all()


def test_memory_layouts():
  x = torch.randn((37, 50), device="cuda")
  exact = _norm([x])
  room = torch.full((37, 100), 1e9, device="cuda")
  room[:, ::2] = x
  odd = torch.cat([x.new_zeros(1), x.reshape(-1)]).bfloat16()[1:]
  for view in (x, x.t(), room[:, ::2], torch._neg_view(x),  # pylint: disable=protected-access
               x.view(37, 5, 10).permute(1, 2, 0), x.expand(1, 37, 50)):
    _near(dense.gradient_norm([view]), exact)
  _near(dense.gradient_norm([x[:1].expand(9, 50)]), 3 * _norm([x[:1]]), 2)
  _near(dense.gradient_norm([odd]), _norm([odd]))
  _near(dense.gradient_norm([x, x]), math.sqrt(2) * exact)
  zero = torch._efficientzerotensor((5,), device="cuda")  # pylint: disable=protected-access
  assert float(dense.gradient_norm([zero])) == 0
  # Scaled where they are, whatever the order of their dimensions.
  y = x.clone()
  dense.clip_gradients([y.t()], exact / 2)
  assert ((y - x / 2).abs() <= 2 * STEP * x.abs()).all()
  for bad in ([room[:, ::2]], [torch._neg_view(y)], [zero],  # pylint: disable=protected-access
              [y[:1].expand(9, 50)], [y, y], [y, y[3:]]):
    before = y.clone()
    with pytest.raises(ValueError):
      dense.clip_gradients(bad, exact / 4)
    assert torch.equal(before, y)


def test_neighbours_stay_as_they_were():
  room = torch.ones(10_000, dtype=torch.bfloat16, device="cuda")
  dense.clip_gradients([room[3:4099], room[4100:9001]], 1e-3)
  assert (room[:3] == 1).all() and room[4099] == 1 and (room[9001:] == 1).all()
  assert (room[3:4099] < 1).all() and (room[4100:9001] < 1).all()


def test_autograd_knows_of_clipped_gradients():
  g, x = torch.ones(5, device="cuda"), torch.ones(5, device="cuda")
  y = (x.requires_grad_() * g).sum()
  dense.clip_gradients([g], 1.0)
  with pytest.raises(RuntimeError):
    y.backward()


def test_factor_scales_adamws_step():
  """A clipped step through grad_scale is the step with clipped gradients: the
  factor is a power of two here, so both round alike."""
  p = _tensors([1000, 77], [torch.float32], 1)
  q = [t.clone() for t in p]
  grads = [torch.full((1000,), 2.0, device="cuda"),
           torch.zeros(77, device="cuda")]
  grads[1][:24] = 2.0  # norm 64
  norm, factor = dense.gradient_norm(grads, max_norm=8.0)
  assert float(norm) == 64 and float(factor) == 0.125
  a, b = dense.init_adamw_state(p), dense.init_adamw_state(q)
  dense.adamw_update(p, grads, a, learning_rate=0.1, grad_scale=factor)
  dense.clip_gradients(grads, 8.0)
  dense.adamw_update(q, grads, b, learning_rate=0.1)
  for x, y in zip([*p, a.m, a.v], [*q, b.m, b.v]):
    assert torch.equal(x, y)


def test_repeated_calls_agree():
  tensors = _tensors([3_000_001, 999], TYPES)
  first = float(dense.gradient_norm(tensors))
  assert all(float(dense.gradient_norm(tensors)) == first for _ in range(5))


def test_refusals():
  x = torch.ones(8, device="cuda")
  for call in (dense.gradient_norm,
               lambda g, max_norm=1.0: dense.clip_gradients(g, max_norm)):
    for bad in ([x.double()], [x.cpu()], [x.to_sparse()], [1.0], [x.int()]):
      with pytest.raises(ValueError):
        call(bad)
    for limit in (-1.0, math.nan):
      with pytest.raises(ValueError):
        call([x], max_norm=limit)
    with pytest.raises(TypeError):
      call([x], max_norm="1")
  with pytest.raises(ValueError):
    dense.clip_gradients([x], None)
  assert (x == 1).all()
