"""Dense operators (lib/nn/dense.py) on more tokens, columns and values than one
launch has threads for (2^32 less one).

Where the arithmetic is the same as in a small call, the small call's results
are expected bit for bit. Sums over a row of n values are added by 1024 lanes
one after another: off by at most (n / 1024 + 64) u of the magnitudes, u being
float32's unit roundoff.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

U = 2.0**-24


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


def test_tokens():
  """8 lanes a token, 2^29 tokens: 2^32 lanes."""
  _need(24)
  n, experts = 2**29 + 37, 5
  ids = torch.randint(-1, experts, (n,), dtype=torch.int32, device="cuda")
  order = dense.sort_by_expert(ids, experts)
  kept = int(order.offsets[-1])
  assert kept == int((ids >= 0).sum())
  x = (torch.arange(n, dtype=torch.int32, device="cuda") % 251).to(
      torch.bfloat16)[:, None]
  rows = dense.tokens_to_experts(x, order)
  assert not rows[kept:].any()
  back = dense.tokens_from_experts(rows, None, order)
  expected = x * (ids >= 0)[:, None]
  assert torch.equal(back, expected)
  # Every row of an expert is from a token that chose it.
  for e in range(experts):
    a, b = int(order.offsets[e]), int(order.offsets[e + 1])
    at = order.sources[a:b].long()
    assert (ids[at] == e).all()
    assert torch.equal(rows[a:b, 0], x[at, 0])
  del rows, at
  drows, _ = dense.tokens_from_experts_grad(x, back, None, order)
  assert not drows[kept:].any()
  assert torch.equal(dense.tokens_to_experts_grad(drows, order), expected)


def test_columns():
  """Weights' gradients of 2^27 columns: 32 columns a work-group of 1024."""
  _need(48)
  rows, dim = 2, 2**27 + 40
  g = torch.Generator(device="cuda").manual_seed(3)
  x = torch.randn((rows, dim), device="cuda", generator=g)
  dy = torch.randn((rows, dim), device="cuda", generator=g)
  mean = x.double().mean(-1).float()
  rstd = x.double().var(-1, correction=0).rsqrt().float()
  dx, _, db = dense.layer_norm_grad(dy, x, mean, rstd)
  _, dw, _ = dense.layer_norm_grad(dy, x, mean, rstd,
                                   torch.ones(dim, device="cuda"),
                                   with_bias=False)
  exact = dy[0].double() + dy[1].double()
  assert ((db - exact).abs() <= 2 * U * (dy[0].abs() + dy[1].abs())).all()
  xhat = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
  part = xhat * dy
  assert ((dw - part.sum(0)).abs() <= 8 * U * part.abs().sum(0)).all()
  sums = dim / 1024 + 64
  for r in range(rows):
    h, along = dy[r].double(), part[r].mean()
    exact = (h - h.mean() - xhat[r] * along) * rstd[r].double()
    tol = U * exact.abs() + rstd[r].double() * U * (
        8 * (h.abs() + (xhat[r] * along).abs()) + sums * (
            h.abs().mean() + xhat[r].abs() * part[r].abs().mean()))
    assert ((dx[r] - exact).abs() <= tol).all()


def test_weights():
  """A weight of more than 2^34 values (1024 a work-group of 256), with a
  small one after it."""
  n = (2**32 // 256) * 1024 + 3 * 1024 + 77
  _need(150)
  tail = 8 * 1024
  cut = n - n % 256 - tail
  g = torch.Generator(device="cuda").manual_seed(4)
  p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
  grad = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
  p[cut:] = torch.randn(n - cut, device="cuda", generator=g)
  grad[cut:] = torch.randn(n - cut, device="cuda", generator=g)
  q = torch.randn(1000, device="cuda", generator=g)
  dq = torch.randn(1000, device="cuda", generator=g)
  # The same values as tensors of their own: blocks begin where they do above.
  small = [p[:512].clone(), p[cut:].clone(), q.clone()]
  small_grads = [grad[:512].clone(), grad[cut:].clone(), dq]
  states = []
  for params, grads in (([p, q], [grad, dq]), (small, small_grads)):
    state = dense.init_adamw_state(params, state_bits=8)
    for _ in range(2):
      dense.adamw_update(params, grads, state, learning_rate=0.1)
    states.append(state)
  big, ref = states
  first = p[0].item()
  assert small[0].eq(first).all() and first != 1.0
  step = 2**30
  for at in range(0, cut, step):
    assert p[at:min(at + step, cut)].eq(first).all()
  assert torch.equal(p[cut:], small[1])
  assert torch.equal(q, small[2])
  del p, grad
  torch.cuda.empty_cache()
  moments = dense.adamw_moments(ref)
  for i, name in enumerate(("m", "v")):
    for at in range(0, cut, step):
      codes = getattr(big, name)[at:min(at + step, cut)]
      assert codes.eq(getattr(ref, name)[0]).all()
    assert torch.equal(getattr(big, name)[cut:], getattr(ref, name)[512:])
    assert torch.equal(getattr(big, name + "_scale")[cut // 256:],
                       getattr(ref, name + "_scale")[2:])
    del codes
  decoded = dense.adamw_moments(big)
  for i in range(2):
    for at in range(0, cut, step):
      assert decoded[i][at:min(at + step, cut)].eq(moments[i][0]).all()
    assert torch.equal(decoded[i][cut:], moments[i][512:])
