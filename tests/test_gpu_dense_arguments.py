"""What a tensor's memory does not say: the dense operators (lib/nn/dense.py) on
views that are negated when read, zeros that were never written, tensors that
are not dense, tensors that share memory, and autograd's view of weights that
were written."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _rand(*shape, seed=0):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return torch.randn(shape, device="cuda", generator=g)


def _same(got, expected):
  for a, b in zip(got, expected, strict=True):
    assert (a is None and b is None) or torch.equal(a, b)


VIEWS = {
    # The same values, and a tensor whose memory holds others.
    "negated": (lambda x: -x, torch._neg_view),  # pylint: disable=protected-access
    "zeros": (torch.zeros_like,
              lambda x: torch._efficientzerotensor(  # pylint: disable=protected-access
                  x.shape, dtype=x.dtype, device=x.device)),
}


@pytest.mark.parametrize("kind", VIEWS)
def test_values_are_not_in_memory(kind):
  plain, lazy = VIEWS[kind]
  x, dy = _rand(9, 24), _rand(9, 24, seed=1)
  w, b = _rand(24, seed=2), _rand(24, seed=3)
  expected = dense.layer_norm(plain(x), plain(w), plain(b), return_stats=True)
  _same(dense.layer_norm(lazy(x), lazy(w), lazy(b), return_stats=True),
        expected)
  mean, rstd = _rand(9, seed=4), _rand(9, seed=5)
  _same(dense.layer_norm_grad(*map(lazy, (dy, x, mean, rstd, w))),
        dense.layer_norm_grad(*map(plain, (dy, x, mean, rstd, w))))

  ids = (torch.arange(18, device="cuda") % 5).view(9, 2)
  order = dense.sort_by_expert(plain(ids), 4)
  _same(dense.sort_by_expert(lazy(ids), 4), order)
  order = dense.sort_by_expert(ids, 4)
  rows, weights = _rand(18, 24, seed=6), _rand(9, 2, seed=7)
  _same([dense.tokens_to_experts(lazy(x), order),
         dense.tokens_to_experts_grad(lazy(rows), order),
         dense.tokens_from_experts(lazy(rows), lazy(weights), order)],
        [dense.tokens_to_experts(plain(x), order),
         dense.tokens_to_experts_grad(plain(rows), order),
         dense.tokens_from_experts(plain(rows), plain(weights), order)])
  _same(dense.tokens_from_experts_grad(lazy(dy), lazy(rows), lazy(weights),
                                       order),
        dense.tokens_from_experts_grad(plain(dy), plain(rows), plain(weights),
                                       order))

  p, q = _rand(300, seed=8), _rand(300, seed=8)
  for params, grad in ((p, lazy(_rand(300))), (q, plain(_rand(300)))):
    dense.adamw_update([params], [grad], dense.init_adamw_state([params]),
                       learning_rate=0.1)
  assert torch.equal(p, q)
  with pytest.raises(ValueError):
    dense.init_adamw_state([lazy(p)])
  with pytest.raises(ValueError):
    dense.adamw_update([p], [q], dense.init_adamw_state([p]),
                       learning_rate=0.1, copies=[lazy(p.bfloat16())])


@pytest.mark.parametrize("dim", [1, 24])
def test_autograd_hands_over_negated_gradients(dim):
  """The gradient of a conjugate's imaginary part is such a view."""
  x, a = _rand(9, dim), _rand(9, dim, seed=1)
  w = _rand(dim, seed=2)

  def grads(joined):
    leaf, weight = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = dense.layer_norm(leaf, weight)
    return torch.autograd.grad(joined(y), [leaf, weight])

  factor = torch.complex(a, 2 * a)
  _same(grads(lambda y: (torch.complex(a, y).conj() * factor).real.sum()),
        grads(lambda y: (y * 2 * a).sum()))


def test_sparse_tensors_are_refused():
  x = _rand(8, 8)
  sparse = x.to_sparse()
  order = dense.sort_by_expert(torch.zeros(8, dtype=torch.int64,
                                           device="cuda"), 2)
  state = dense.init_adamw_state([x])
  for call in (lambda: dense.layer_norm(sparse),
               lambda: dense.layer_norm(x.to_sparse_csr()),
               lambda: dense.tokens_to_experts(sparse, order),
               lambda: dense.init_adamw_state([sparse]),
               lambda: dense.adamw_update([x], [sparse], state,
                                          learning_rate=0.1)):
    with pytest.raises(ValueError):
      call()


@pytest.mark.parametrize("inference", [False, True])
def test_autograd_knows_of_updated_weights(inference):
  with torch.inference_mode(inference):
    p, other, copy = _rand(300), _rand(300), _rand(300).bfloat16()
  state = dense.init_adamw_state([p, other])
  if inference:
    dense.adamw_update([p, other], [_rand(300), None], state,
                       learning_rate=0.1, copies=[copy, None])
    assert torch.equal(copy, p.bfloat16())
    return
  x = _rand(300).requires_grad_()
  stale, fresh = (x * p).sum(), (x * other).sum()
  stale_copy = (x * copy).sum()
  dense.adamw_update([p, other], [_rand(300), None], state, learning_rate=0.1,
                     copies=[copy, None])
  fresh.backward()
  assert torch.equal(x.grad, other)
  for y in (stale, stale_copy):
    with pytest.raises(RuntimeError):
      y.backward()


def test_copies_share_no_memory():
  p, q = _rand(300), _rand(300, seed=1)
  half = _rand(300, seed=2).bfloat16()
  room = torch.zeros(400, dtype=torch.bfloat16, device="cuda")
  g = _rand(300, seed=3)
  for params, copies in (([p, q], [room[:300], room[100:]]),
                         ([p, half], [half, None]),
                         ([p, q], [q.view(torch.bfloat16)[:300], None]),
                         ([p], [p.view(torch.bfloat16)[:300]])):
    before = [x.clone() for x in params]
    state = dense.init_adamw_state(params)
    with pytest.raises(ValueError):
      dense.adamw_update(params, [g] * len(params), state, learning_rate=0.1,
                         copies=copies)
    _same(params, before)
  # A bfloat16 weight is its own copy.
  expected = half.clone()
  for w, copies in ((half, [half]), (expected, None)):
    dense.adamw_update([w], [g], dense.init_adamw_state([w]),
                       learning_rate=0.1, copies=copies)
  assert torch.equal(half, expected)
