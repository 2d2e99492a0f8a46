"""The experts' products (lib/nn/dense.py) against plain products in 64 bits.

Two kinds of values. Small whole numbers: every product and every sum is exact
in float32, so results are expected bit for bit, rounded once to their type.
Normal values: a sum of n products is off by at most n roundings of partial
sums, each below the sum of the magnitudes; the matrix instructions' additions
are taken to round by a whole step (2u, u = 2^-24, the unit roundoff), and the
result's own rounding adds half a step of its type.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _order(offsets):
  return dense.ExpertOrder(None, None, torch.tensor(
      offsets, dtype=torch.int32, device="cuda"))


def _offsets(counts, dropped=0):
  """(offsets, rows in all)."""
  out = [0]
  for c in counts:
    out.append(out[-1] + c)
  return out, out[-1] + dropped


def _values(shape, dtype, seed, whole):
  g = torch.Generator(device="cuda").manual_seed(seed)
  if whole:
    x = torch.randint(-3, 4, shape, device="cuda", generator=g)
  else:
    x = torch.randn(shape, device="cuda", generator=g)
  return x.to(dtype)


def _expected(x, w, dy, offsets):
  """(y, rows' gradient, weights' gradient) in 64 bits, on the CPU."""
  x, w = x.double().cpu(), w.double().cpu()
  y = torch.zeros((x.shape[0], w.shape[2]), dtype=torch.float64)
  dx, dw = torch.zeros_like(x), torch.zeros_like(w)
  dy = dy.double().cpu()
  for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
    y[a:b] = x[a:b] @ w[e]
    dx[a:b] = dy[a:b] @ w[e].t()
    dw[e] = x[a:b].t() @ dy[a:b]
  return y, dx, dw


def _check(got, exact, size, terms, whole):
  """size: the sum of the terms' magnitudes."""
  assert got.shape == exact.shape
  if whole:
    assert torch.equal(got.cpu(), exact.to(got.dtype))
    return
  bound = (2 * U * (terms + 2) * size +
           torch.finfo(got.dtype).eps / 2 * exact.abs() + 1e-7 * (
               got.dtype == torch.float16))
  assert ((got.double().cpu() - exact).abs() <= bound).all()


def _run(x, w, dy, offsets, whole):
  order = _order(offsets)
  # What no expert has is not read.
  x, dy = x.clone(memory_format=torch.preserve_format), dy.clone()
  x[offsets[-1]:] = float("nan")
  dy[offsets[-1]:] = float("inf")
  y = dense.expert_matmul(x, w, order)
  dx, dw = dense.expert_matmul_grad(dy, x, w, order)
  x[offsets[-1]:] = 0
  dy[offsets[-1]:] = 0
  exact = _expected(x, w, dy, offsets)
  sizes = _expected(x.abs(), w.abs(), dy.abs(), offsets)
  most = max([b - a for a, b in zip(offsets, offsets[1:])])
  for got, e, s, terms in zip((y, dx, dw), exact, sizes,
                              (w.shape[1], w.shape[2], most)):
    assert got.dtype == x.dtype
    _check(got, e, s, terms, whole)


COUNTS = {
    "one_row": ([1], 0),
    "single_rows": ([1] * 8, 0),
    "some_empty": ([0, 5, 0, 0, 17, 1, 0], 3),
    "all_dropped": ([0, 0, 0], 9),
    "whole_tiles": ([128, 256, 384], 0),
    "ragged": ([127, 1, 129, 300, 64], 5),
    "one_large": ([3, 1500, 2], 40),
    "many_experts": ([i % 3 for i in range(1024)], 1),
}


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("inner,outer", [(64, 128), (72, 40), (100, 36),
                                         (33, 7)])
def test_rows_of_experts(counts, inner, outer, dtype, whole):
  offsets, n = _offsets(*COUNTS[counts])
  experts = len(offsets) - 1
  x = _values((n, inner), dtype, 1, whole)
  w = _values((experts, inner, outer), dtype, 2, whole)
  dy = _values((n, outer), dtype, 3, whole)
  _run(x, w, dy, offsets, whole)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [
    (1, 1), (1, 200), (200, 1), (2, 3), (8, 8), (64, 64), (65, 63), (127, 129),
    (128, 256), (192, 320), (256, 264), (264, 512), (515, 130), (1000, 24),
    (16, 1032)])
@pytest.mark.parametrize("stored", ["in_out", "out_in"])
def test_sizes(inner, outer, stored, dtype):
  offsets, n = _offsets([40, 0, 300, 7], 6)
  x = _values((n, inner), dtype, 1, True)
  w = _values((4, inner, outer), dtype, 2, True)
  if stored == "out_in":
    w = w.transpose(1, 2).contiguous().transpose(1, 2)
  dy = _values((n, outer), dtype, 3, True)
  _run(x, w, dy, offsets, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stored", ["in_out", "out_in"])
def test_many_rows(stored, dtype):
  """The largest tiles, more of them than CUs."""
  offsets, n = _offsets([5000, 0, 9000, 2467], 100)
  inner, outer = 520, 776
  x = _values((n, inner), dtype, 1, True)
  w = _values((4, inner, outer), dtype, 2, True)
  if stored == "out_in":
    w = w.transpose(1, 2).contiguous().transpose(1, 2)
  dy = _values((n, outer), dtype, 3, True)
  _run(x, w, dy, offsets, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stored", ["in_out", "out_in"])
@pytest.mark.parametrize("inner,outer", [(4096, 40), (1100, 128), (2051, 130),
                                         (1999, 3), (1024, 256)])
def test_long_sums_of_few_rows(inner, outer, stored, dtype):
  """Cut along the sum, forwards and, with inner and outer changed about,
  backwards; some parts are shorter or have nothing."""
  offsets, n = _offsets([40, 0, 3, 61], 6)
  x = _values((n, inner), dtype, 1, True)
  w = _values((4, inner, outer), dtype, 2, True)
  if stored == "out_in":
    w = w.transpose(1, 2).contiguous().transpose(1, 2)
  dy = _values((n, outer), dtype, 3, True)
  # float16 ends at 65504: sums of 4096 products of 9 stay below.
  _run(x, w, dy, offsets, True)
  _run(dy, w.transpose(1, 2), x, offsets, True)


def _strided(x, how):
  """The same values in other memory."""
  if how == "padded_rows":
    room = torch.full((*x.shape[:-1], x.shape[-1] + 8), float("nan"),
                      dtype=x.dtype, device="cuda")
    room[..., :x.shape[-1]] = x
    return room[..., :x.shape[-1]]
  if how == "odd_rows":
    room = torch.full((*x.shape[:-1], x.shape[-1] + 3), float("nan"),
                      dtype=x.dtype, device="cuda")
    room[..., 1:x.shape[-1] + 1] = x
    return room[..., 1:x.shape[-1] + 1]
  if how == "every_other":
    room = torch.full((*x.shape[:-1], 2 * x.shape[-1]), float("nan"),
                      dtype=x.dtype, device="cuda")
    room[..., ::2] = x
    return room[..., ::2]
  if how == "odd_start":
    room = torch.full((x.numel() + 1,), float("nan"), dtype=x.dtype,
                      device="cuda")
    room[1:] = x.reshape(-1)
    return room[1:].view(x.shape)
  dims = list(range(x.dim()))[::-1]  # "reversed": columns first in memory
  return x.permute(dims).contiguous().permute(dims)


@pytest.mark.parametrize("how", ["padded_rows", "odd_rows", "every_other",
                                 "odd_start", "reversed"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_memory_layouts(how, dtype):
  offsets, n = _offsets([140, 3, 0, 61], 2)
  x, w = _values((n, 72), dtype, 1, True), _values((4, 72, 48), dtype, 2, True)
  dy = _values((n, 48), dtype, 3, True)
  order = _order(offsets)
  y = dense.expert_matmul(x, w, order)
  dx, dw = dense.expert_matmul_grad(dy, x, w, order)
  sx, sw, sdy = _strided(x, how), _strided(w, how), _strided(dy, how)
  assert torch.equal(dense.expert_matmul(sx, sw, order), y)
  got = dense.expert_matmul_grad(sdy, sx, sw, order)
  assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
  # Operands that are one value or one row in memory.
  e = x[:1, :1].expand(n, 72)
  assert torch.equal(dense.expert_matmul(e, w, order),
                     dense.expert_matmul(e.contiguous(), w, order))
  one = w[:1].expand(4, -1, -1)
  assert torch.equal(dense.expert_matmul(x, one, order),
                     dense.expert_matmul(x, one.contiguous(), order))


def test_weights_gradient_is_laid_out_as_the_weights():
  offsets, n = _offsets([10, 20])
  x, dy = _values((n, 24), torch.float32, 1, True), _values(
      (n, 40), torch.float32, 2, True)
  w = _values((2, 40, 24), torch.float32, 3, True)
  _, dw = dense.expert_matmul_grad(dy, x, w.transpose(1, 2), _order(offsets))
  assert dw.transpose(1, 2).is_contiguous()
  _, dw = dense.expert_matmul_grad(dy, x, w.transpose(1, 2).contiguous(),
                                   _order(offsets))
  assert dw.is_contiguous()


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(dtype):
  """An infinity or a NaN reaches its own row, and its expert's weights'
  gradient, alone."""
  offsets, n = _offsets([150, 40, 150], 4)
  x, w = _values((n, 96), dtype, 1, True), _values((3, 96, 80), dtype, 2, True)
  w[w == 0] = 1
  dy = _values((n, 80), dtype, 3, True)
  order = _order(offsets)
  y = dense.expert_matmul(x, w, order)
  dx, dw = dense.expert_matmul_grad(dy, x, w, order)
  x[7, 95] = float("inf")
  x[160, 0] = float("nan")
  got = dense.expert_matmul(x, w, order)
  expected = x.double() @ w[0].double()
  assert torch.equal(got[7], expected[7].to(dtype))
  assert got[7].isinf().all() and got[160].isnan().all()
  keep = torch.ones(n, dtype=torch.bool, device="cuda")
  keep[[7, 160]] = False
  assert torch.equal(got[keep], y[keep])
  dy[339, 3] = float("nan")
  gx, gw = dense.expert_matmul_grad(dy, x, w, order)
  keep[:] = True
  keep[339] = False
  assert torch.equal(gx[keep], dx[keep]) and gx[339].isnan().all()
  assert torch.equal(gw[0, :95], dw[0, :95])
  assert not gw[0, 95].isfinite().all()
  assert torch.equal(gw[1, 1:], dw[1, 1:]) and gw[1, 0].isnan().all()
  assert gw[2, :, 3].isnan().all()
  assert torch.equal(gw[2, :, 4:], dw[2, :, 4:])


def test_no_rows():
  w = _values((3, 8, 16), torch.bfloat16, 1, True)
  x = torch.empty((0, 8), dtype=torch.bfloat16, device="cuda")
  order = _order([0, 0, 0, 0])
  assert dense.expert_matmul(x, w, order).shape == (0, 16)
  dx, dw = dense.expert_matmul_grad(x.new_empty((0, 16)), x, w, order)
  assert dx.shape == (0, 8) and not dw.any() and dw.shape == w.shape


def test_only_what_is_wanted():
  offsets, n = _offsets([10, 20])
  x, w = _values((n, 8), torch.float32, 1, True), _values(
      (2, 8, 8), torch.float32, 2, True)
  dx, dw = dense.expert_matmul_grad(x, x, w, _order(offsets))
  a = dense.expert_matmul_grad(x, x, w, _order(offsets), with_rows=False)
  b = dense.expert_matmul_grad(x, x, w, _order(offsets), with_weights=False)
  assert a[0] is None and torch.equal(a[1], dw)
  assert b[1] is None and torch.equal(b[0], dx)


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(dtype):
  offsets, n = _offsets([33, 0, 70], 5)
  x, w = _values((n, 40), dtype, 1, False), _values((3, 40, 24), dtype, 2,
                                                    False)
  dy = _values((n, 24), dtype, 3, False)
  order = _order(offsets)
  lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
  y = dense.expert_matmul(lx, lw, order)
  assert torch.equal(y.detach(), dense.expert_matmul(x, w, order))
  dx, dw = dense.expert_matmul_grad(dy, x, w, order)
  got = torch.autograd.grad(y, [lx, lw], dy, retain_graph=True)
  assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
  assert torch.equal(torch.autograd.grad(y, lw, dy, retain_graph=True)[0], dw)
  # A scalar's gradient is one value in memory.
  one, _ = torch.autograd.grad(y.sum(), [lx, lw])
  assert torch.equal(one, dense.expert_matmul_grad(
      torch.ones_like(dy), x, w, order)[0])


def test_gradient_against_differences():
  """Whole numbers and steps of a whole: (f(x + d) - f(x - d)) / 2 is exact
  where f is linear."""
  offsets, n = _offsets([30, 9], 1)
  x, w = _values((n, 24), torch.float32, 1, True), _values(
      (2, 24, 16), torch.float32, 2, True)
  c = _values((n, 16), torch.float32, 3, True)
  order = _order(offsets)
  f = lambda x, w: (dense.expert_matmul(x, w, order) * c).sum().item()
  dx, dw = dense.expert_matmul_grad(c, x, w, order)
  for at in [(0, 0), (29, 23), (30, 5), (38, 11), (39, 3)]:
    d = torch.zeros_like(x)
    d[at] = 1
    assert (f(x + d, w) - f(x - d, w)) / 2 == dx[at].item()
  for at in [(0, 0, 0), (0, 23, 15), (1, 11, 7)]:
    d = torch.zeros_like(w)
    d[at] = 1
    assert (f(x, w + d) - f(x, w - d)) / 2 == dw[at].item()


def test_repeated_calls_agree():
  offsets, n = _offsets([3000, 11, 1200], 5)
  for dtype in TYPES:
    x, w = _values((n, 136), dtype, 1, False), _values((3, 136, 72), dtype, 2,
                                                       False)
    dy = _values((n, 72), dtype, 3, False)
    order = _order(offsets)
    first = (dense.expert_matmul(x, w, order),
             *dense.expert_matmul_grad(dy, x, w, order))
    for _ in range(3):
      again = (dense.expert_matmul(x, w, order),
               *dense.expert_matmul_grad(dy, x, w, order))
      for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_offsets_that_do_not_fit_reach_no_memory():
  """Offsets past the rows, negative ones, falling ones: whatever comes out,
  memory outside the result stays as it was."""
  n = 50
  x, w = _values((n, 16), torch.float32, 1, True), _values(
      (3, 16, 8), torch.float32, 2, True)
  for offsets in ([0, 20, 40, 5000], [-100, 20, 40, 50], [0, 40, 10, 50],
                  [60, 70, 80, 90]):
    y = dense.expert_matmul(x, w, _order(offsets))
    dx, dw = dense.expert_matmul_grad(y, x, w, _order(offsets))
    assert y.shape == (n, 8) and dx.shape == x.shape and dw.shape == w.shape
  y = dense.expert_matmul(x, w, _order([0, 20, 40, 5000]))
  assert torch.equal(y, dense.expert_matmul(x, w, _order([0, 20, 40, 50])))


def test_offsets_that_do_not_fit_in_pieces():
  """The weights' gradient in pieces: segments that overlap have more pieces
  than there are places for."""
  n, experts = 20_000, 9
  x, dy = _values((n, 16), torch.float32, 1, True), _values(
      (n, 8), torch.float32, 2, True)
  w = _values((experts, 16, 8), torch.float32, 3, True)
  good = _order([i * n // experts for i in range(experts + 1)])
  expected = dense.expert_matmul_grad(dy, x, w, good)
  for offsets in ([0, n] * 5, [n, 0] * 5, [-5] * 9 + [2**31 - 1]):
    dx, dw = dense.expert_matmul_grad(dy, x, w, _order(offsets))
    assert dx.shape == x.shape and dw.shape == w.shape
  for a, b in zip(dense.expert_matmul_grad(dy, x, w, good), expected):
    assert torch.equal(a, b)


def test_refusals():
  x = torch.zeros((6, 8), device="cuda")
  w = torch.zeros((2, 8, 4), device="cuda")
  order = _order([0, 3, 6])
  dense.expert_matmul(x, w, order)
  off = order.offsets
  for bad in (
      lambda: dense.expert_matmul(x.double(), w.double(), order),
      lambda: dense.expert_matmul(x, w.bfloat16(), order),
      lambda: dense.expert_matmul(x[0], w, order),
      lambda: dense.expert_matmul(x[:, :0], w[:, :0], order),
      lambda: dense.expert_matmul(x, w[0], order),
      lambda: dense.expert_matmul(x, w[:1], order),
      lambda: dense.expert_matmul(x, w[:, :7], order),
      lambda: dense.expert_matmul(x, w[:, :, :0], order),
      lambda: dense.expert_matmul(x.cpu(), w, order),
      lambda: dense.expert_matmul(x, w.cpu(), order),
      lambda: dense.expert_matmul(x.to_sparse(), w, order),
      lambda: dense.expert_matmul(x, w, order._replace(offsets=off.long())),
      lambda: dense.expert_matmul(x, w, order._replace(offsets=off[:1])),
      lambda: dense.expert_matmul(x, w, order._replace(offsets=off.cpu())),
      lambda: dense.expert_matmul([1.0], w, order),
      lambda: dense.expert_matmul_grad(x, x, w, order),
      lambda: dense.expert_matmul_grad(x[:5, :4], x, w, order),
      lambda: dense.expert_matmul_grad(x[:, :4].half(), x, w, order)):
    with pytest.raises(ValueError):
      bad()
