"""Tokens sorted by expert and back (lib/nn/dense.py) against the definitions:
orders and copies exactly, sums in 64 bits.

Tolerances. u is float32's unit roundoff, uo the result's. A sum over k choices
is off by at most (k + 1) u times the sum of magnitudes; an inner product over
dim values, added by up to 64 lanes, by (dim / 64 + 8) u of it (dim u where a
lane has the row). Products of one weight and one value round once.
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

U = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8,
         torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _ids(rng, shape, experts, dtype=np.int64, dropped=0.1, skew=1.0):
  p = rng.random(experts) ** (1 + skew)
  ids = rng.choice(experts, size=shape, p=p / p.sum()).astype(dtype)
  gone = rng.random(shape) < dropped
  ids[gone] = rng.choice([-1, experts, experts + 7, -(2**31), 2**31 - 1],
                         size=int(gone.sum()))
  return ids


def _expected_order(ids, experts):
  flat = ids.reshape(-1).astype(np.int64)
  key = np.where((flat >= 0) & (flat < experts), flat, experts)
  sources = np.argsort(key, kind="stable")
  positions = np.empty(flat.size, np.int64)
  positions[sources] = np.arange(flat.size)
  offsets = np.searchsorted(key[sources], np.arange(experts + 1))
  return positions.reshape(ids.shape), sources, offsets


def _check_order(ids, experts):
  order = dense.sort_by_expert(torch.from_numpy(ids).cuda(), experts)
  for got, expected in zip(order, _expected_order(ids, experts)):
    assert got.dtype == torch.int32
    assert np.array_equal(got.cpu().numpy(), expected)
  return order


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
@pytest.mark.parametrize("experts", [1, 2, 7, 64, 65, 255, 1021, 1022, 1023,
                                     1024])
def test_sort(experts, dtype):
  rng = np.random.default_rng(experts)
  # Both sides of the sizes where one work-group and a tile end.
  for shape in [(0, 2), (1, 1), (1, 3), (63,), (64, 1), (65, 1), (1000, 2),
                (4096, 2), (8193, 1), (2731, 3), (5000, 8), (20011, 3)]:
    print(experts, dtype, shape, flush=True)
    _check_order(_ids(rng, shape, experts, dtype), experts)


@pytest.mark.parametrize("n", [8192, 300_000, 5_000_000])
def test_sort_extremes(n):
  """Every choice of one expert; every choice dropped; already in order and
  in reverse; more ids than the tiles of the base size cover."""
  for ids in (np.full(n, 3), np.full(n, -1), np.arange(n) * 8 // n,
              7 - np.arange(n) * 8 // n, np.arange(n) % 8):
    _check_order(ids.astype(np.int64), 8)


def test_sort_takes_any_strides():
  rng = np.random.default_rng(5)
  ids = _ids(rng, (300, 6), 11)
  t = torch.from_numpy(ids).cuda()
  for view, host in ((t[:, ::2], ids[:, ::2]), (t.t(), ids.T)):
    got = dense.sort_by_expert(view, 11)
    expected = _expected_order(np.ascontiguousarray(host), 11)
    for a, b in zip(got, expected):
      assert np.array_equal(a.cpu().numpy(), b)


def _case(tokens, choices, experts, dim, dtype, seed=0, dropped=0.2):
  rng = np.random.default_rng(seed)
  shape = (tokens, choices) if choices else (tokens,)
  ids = torch.from_numpy(_ids(rng, shape, experts, dropped=dropped)).cuda()
  order = dense.sort_by_expert(ids, experts)
  g = torch.Generator(device="cuda").manual_seed(seed)
  new = lambda *s: torch.randn(s, device="cuda", generator=g).to(dtype)
  n = ids.numel()
  x, rows, dy = new(tokens, dim), new(n, dim), new(tokens, dim)
  weights = torch.rand(shape, device="cuda", generator=g)
  return order, x, rows, dy, weights


def _picked(rows, order):
  """[tokens, choices, dim] in 64 bits, zero where dropped, and where kept."""
  pos = order.positions.long()
  pos = pos if pos.dim() == 2 else pos.unsqueeze(1)
  kept = pos < order.offsets[-1]
  return torch.where(kept.unsqueeze(2), rows.double()[pos], 0.0), kept


def _check_all(order, x, rows, dy, weights):
  dtype, dim = rows.dtype, rows.shape[1]
  kept_rows = int(order.offsets[-1])
  k = order.positions.numel() // max(1, order.positions.shape[0])
  # To the experts: a copy.
  got = dense.tokens_to_experts(x, order)
  expected = x[order.sources.long() // max(k, 1)].clone()
  expected[kept_rows:] = 0
  assert got.dtype == dtype and torch.equal(got, expected)
  # What dropped rows hold is never read.
  dirty = rows.clone()
  dirty[kept_rows:] = float("nan")
  picked, kept = _picked(rows, order)
  exact = picked.sum(1)
  tol = ROUND[dtype] * exact.abs() + (k + 1) * U * picked.abs().sum(1) + (
      TINY[dtype])
  got = dense.tokens_to_experts_grad(dirty, order)
  assert got.dtype == dtype
  assert ((got.double() - exact).abs() <= tol).all()
  # Back from the experts.
  for w in (weights, weights.to(dtype), None):
    wd = (torch.ones_like(kept, dtype=torch.float64) if w is None else
          w.double().view(kept.shape))
    parts = picked * wd.unsqueeze(2)
    exact = parts.sum(1)
    tol = ROUND[dtype] * exact.abs() + (k + 1) * U * parts.abs().sum(1) + (
        TINY[dtype])
    got = dense.tokens_from_experts(dirty, w, order)
    assert got.dtype == dtype and got.shape == dy.shape
    assert ((got.double() - exact).abs() <= tol).all()
    drows, dw = dense.tokens_from_experts_grad(dy, dirty, w, order)
    exact = torch.zeros(rows.shape, dtype=torch.float64, device="cuda")
    exact[order.positions.long().view(-1)] = (
        torch.where(kept, wd, 0.0).unsqueeze(2) *
        dy.double().unsqueeze(1)).view(-1, dim)
    assert drows.dtype == dtype
    assert ((drows.double() - exact).abs() <= (ROUND[dtype] + U) * exact.abs() +
            TINY[dtype]).all()
    assert (drows[kept_rows:] == 0).all()
    if w is None:
      assert dw is None
      continue
    parts = picked * dy.double().unsqueeze(1)
    exact = parts.sum(2).view(w.shape)
    tol = ROUND[w.dtype] * exact.abs() + (dim + 8) * U * (
        parts.abs().sum(2).view(w.shape)) + TINY[w.dtype]
    assert dw.dtype == w.dtype
    assert ((dw.double() - exact).abs() <= tol).all()


@pytest.mark.parametrize("dtype", list(ROUND), ids=str)
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 6, 8, 12, 64, 100, 127, 128, 132,
                                 256, 511, 520, 1024, 2050, 4096])
def test_rows(dim, dtype):
  print(dim, dtype, flush=True)
  _check_all(*_case(67, 3, 5, dim, dtype, seed=dim))


@pytest.mark.parametrize("choices", [0, 1, 2, 3, 4, 5, 8, 17])
@pytest.mark.parametrize("tokens", [0, 1, 2, 33, 700])
def test_tokens_and_choices(tokens, choices):
  """choices 0: ids of one dimension."""
  _check_all(*_case(tokens, choices, 20, 48, torch.bfloat16, seed=tokens))


@pytest.mark.parametrize("dropped", [0.0, 0.9, 1.0])
def test_dropped(dropped):
  _check_all(*_case(100, 2, 4, 40, torch.float32, dropped=dropped))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_strides(dtype):
  order, x, rows, dy, weights = _case(60, 2, 6, 72, dtype)
  def within(t, at, columns=80):
    wide = torch.zeros((t.shape[0], columns), dtype=dtype, device="cuda")
    wide[:, at:at + t.shape[1]] = t
    return wide[:, at:at + t.shape[1]]
  _check_all(order, within(x, 8), within(rows, 8), within(dy, 8), weights)
  _check_all(order, within(x, 3), within(rows, 1), within(dy, 5), weights)
  _check_all(order, x.t().contiguous().t(), rows.t().contiguous().t(),
             dy.t().contiguous().t(), weights.t().contiguous().t())
  one = dy[:1].expand(dy.shape)
  _check_all(order, x[:1].expand(x.shape), rows, one, weights)


def test_what_dropped_choices_hold_is_not_read():
  """Infinite and undefined weights, rows and tokens of dropped choices."""
  order, x, rows, dy, weights = _case(40, 3, 6, 24, torch.float32, dropped=0.4)
  gone = order.positions >= order.offsets[-1]
  clean = (dense.tokens_from_experts(rows, weights, order),
           dense.tokens_from_experts_grad(dy, rows, weights, order))
  for bad in (float("nan"), float("inf"), -float("inf"),
              torch.finfo(torch.float32).min):
    w, r = weights.clone(), rows.clone()
    w[gone] = bad
    r[int(order.offsets[-1]):] = bad
    assert torch.equal(dense.tokens_from_experts(r, w, order), clean[0])
    got = dense.tokens_from_experts_grad(dy, r, w, order)
    assert torch.equal(got[0], clean[1][0]) and torch.equal(got[1],
                                                            clean[1][1])
    t = x.clone()
    t[gone.all(1)] = bad
    assert torch.equal(dense.tokens_to_experts(t, order),
                       dense.tokens_to_experts(x, order))
  none = dense.sort_by_expert(torch.full((40, 3), -1, device="cuda"), 6)
  assert (dense.tokens_from_experts(rows, weights, none) == 0).all()
  assert (dense.tokens_to_experts_grad(rows, none) == 0).all()


def test_wrong_positions_are_dropped():
  """Positions that no sort gives neither fault nor touch other rows."""
  order, x, rows, dy, weights = _case(20, 2, 4, 16, torch.float32, dropped=0.0)
  pos = order.positions.clone()
  lost = int(pos[3, 1])
  pos[3, 1] = -5
  pos[4, 0] = 2**31 - 1
  bad = dense.ExpertOrder(pos, order.sources, order.offsets)
  got = dense.tokens_from_experts(rows, weights, bad)
  w = weights.clone()
  w[3, 1] = w[4, 0] = 0.0
  expected = dense.tokens_from_experts(rows, w, order)
  assert torch.allclose(got, expected, rtol=1e-6, atol=1e-6)
  assert dense.tokens_to_experts(x, bad).shape == rows.shape
  _, dw = dense.tokens_from_experts_grad(dy, rows, weights, bad)
  assert dw[3, 1] == 0 and dw[4, 0] == 0 and lost >= 0
  many = order.offsets.clone()
  many[-1] = 2**31 - 1
  got = dense.tokens_from_experts(rows, weights,
                                  dense.ExpertOrder(pos, None, many))
  assert torch.equal(got, dense.tokens_from_experts(rows, weights, bad))
  # No choices are kept, by a count that no sort gives either.
  many[-1] = -3
  none = dense.ExpertOrder(order.positions, order.sources, many)
  assert (dense.tokens_from_experts(rows, weights, none) == 0).all()
  assert (dense.tokens_to_experts(x, none) == 0).all()
  drows, dw = dense.tokens_from_experts_grad(dy, rows, weights, none)
  assert (drows == 0).all() and (dw == 0).all()


def test_autograd_and_differences():
  order, x, _, c, weights = _case(30, 2, 4, 12, torch.float32, seed=3)
  x, weights = x.requires_grad_(), weights.requires_grad_()
  rows = dense.tokens_to_experts(x, order)
  y = dense.tokens_from_experts(rows * rows, weights, order)
  (y * c).sum().backward()

  def f(x, w):
    pos = order.positions.long()
    kept = (pos < order.offsets[-1]).double()
    picked = x.unsqueeze(1) * kept.unsqueeze(2)
    return ((picked * picked * w.unsqueeze(2)).sum(1) * c.double()).sum()

  g = torch.Generator(device="cuda").manual_seed(2)
  args = [x.detach().double(), weights.detach().double()]
  for i, grad in enumerate((x.grad, weights.grad)):
    d = torch.randn(args[i].shape, device="cuda", generator=g).double()
    h = 1e-5
    up = [a + h * d if j == i else a for j, a in enumerate(args)]
    down = [a - h * d if j == i else a for j, a in enumerate(args)]
    slope = (f(*up) - f(*down)) / (2 * h)
    along = grad.double() * d
    # f is a quadratic in either: differences are exact up to 1e-16 / h.
    assert (along.sum() - slope).abs() <= 64 * U * along.abs().sum() + 1e-7


def test_gradients_that_nobody_asks_for():
  order, _, rows, dy, weights = _case(30, 2, 4, 12, torch.bfloat16)
  w = weights.clone().requires_grad_()
  dense.tokens_from_experts(rows, w, order).backward(dy)
  assert torch.equal(
      w.grad, dense.tokens_from_experts_grad(dy, rows, weights, order)[1])
  r = rows.clone().requires_grad_()
  dense.tokens_from_experts(r, None, order).backward(dy)
  assert torch.equal(
      r.grad, dense.tokens_from_experts_grad(dy, rows, None, order)[0])


def test_offsets_past_32_bits():
  """Rows whose elements lie past 2^31."""
  tokens, dim = 3, 8
  ids = torch.tensor([[1], [0], [1]], device="cuda")
  order = dense.sort_by_expert(ids, 2)
  stride = 1 << 30
  big = torch.empty(2 * stride + dim, dtype=torch.bfloat16, device="cuda")
  rows = big.as_strided((tokens, dim), (stride, 1))
  values = torch.randn((tokens, dim), device="cuda").bfloat16()
  rows.copy_(values)
  assert torch.equal(dense.tokens_to_experts(rows, order), values[[1, 0, 2]])
  assert torch.equal(dense.tokens_from_experts(rows, None, order),
                     values[[1, 0, 2]])
  drows, dw = dense.tokens_from_experts_grad(
      values, rows, torch.ones((3, 1), device="cuda"), order)
  assert torch.equal(drows, values[[1, 0, 2]])
  exact = (values.double() * values[[1, 0, 2]].double()).sum(1, keepdim=True)
  assert torch.allclose(dw.double(), exact, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dim", [1024, 1023])
def test_more_than_the_caches(dim):
  """Calls of more than 256 MB read their rows past the caches."""
  tokens = 50000
  order, x, rows, _, weights = _case(tokens, 2, 16, dim, torch.bfloat16,
                                     dropped=0.05)
  got = dense.tokens_to_experts(x, order)
  expected = x[order.sources.long() // 2]
  expected[int(order.offsets[-1]):] = 0
  assert torch.equal(got, expected)
  y = dense.tokens_from_experts(rows, weights, order)
  for at in range(0, tokens, 10000):
    part = dense.ExpertOrder(order.positions[at:at + 10000], None,
                             order.offsets)
    picked, kept = _picked(rows, part)
    parts = picked * torch.where(kept, weights[at:at + 10000].double(),
                                 0.0).unsqueeze(2)
    exact = parts.sum(1)
    tol = ROUND[torch.bfloat16] * exact.abs() + 3 * U * parts.abs().sum(1)
    assert ((y[at:at + 10000].double() - exact).abs() <= tol).all()


def test_refusals():
  order, x, rows, dy, weights = _case(20, 2, 4, 16, torch.float32)
  ids = torch.zeros((20, 2), dtype=torch.int64, device="cuda")
  bad = [
      lambda: dense.sort_by_expert(ids.cpu(), 4),
      lambda: dense.sort_by_expert(ids.float(), 4),
      lambda: dense.sort_by_expert(ids.view(1, 20, 2), 4),
      lambda: dense.sort_by_expert(ids, 0),
      lambda: dense.sort_by_expert(ids, 1025),
      lambda: dense.tokens_to_experts(x[:19], order),
      lambda: dense.tokens_to_experts(x[:, :0], order),
      lambda: dense.tokens_to_experts(x.double(), order),
      lambda: dense.tokens_to_experts(x, order._replace(
          positions=order.positions.long())),
      lambda: dense.tokens_to_experts(x, order._replace(
          offsets=order.offsets[:1])),
      lambda: dense.tokens_to_experts_grad(rows[:39], order),
      lambda: dense.tokens_from_experts(rows[:39], weights, order),
      lambda: dense.tokens_from_experts(rows, weights[:, :1], order),
      lambda: dense.tokens_from_experts(rows, weights.double(), order),
      lambda: dense.tokens_from_experts(rows, weights.cpu(), order),
      lambda: dense.tokens_from_experts_grad(dy[:, :8], rows, weights, order),
      lambda: dense.tokens_from_experts_grad(dy.half(), rows, weights, order),
  ]
  for call in bad:
    with pytest.raises(ValueError):
      call()
