"""What the experts' C entries write of an order that no sort made: the rows at
the positions that are in range, and nothing else. A row that no choice has
keeps what it held, and nothing past the rows is touched."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore import _native  # pylint: disable=g-import-not-at-top,wrong-import-position
from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

HELD = 7.0  # what an output holds before the call


class Order(ctypes.Structure):
  _fields_ = [("positions", ctypes.c_void_p), ("offsets", ctypes.c_void_p),
              ("tokens", ctypes.c_int64), ("choices", ctypes.c_int32),
              ("num_experts", ctypes.c_int32)]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _args(x):
  return ctypes.c_void_p(x.data_ptr())


@pytest.mark.parametrize("dim", [5, 16, 130])
def test_rows_that_no_choice_has(dim):
  tokens, choices, experts, past = 20, 2, 4, 3
  n = tokens * choices
  g = torch.Generator(device="cuda").manual_seed(dim)
  ids = torch.randint(0, experts, (tokens, choices), device="cuda", generator=g)
  ids[7] = -1  # dropped by their ids: zeros
  order = dense.sort_by_expert(ids, experts)
  x = torch.randn((tokens, dim), device="cuda", generator=g)
  rows_in = torch.randn((n, dim), device="cuda", generator=g)
  w = torch.rand((tokens, choices), device="cuda", generator=g)
  # Positions out of range, below and above.
  pos = order.positions.clone()
  lost = [int(pos[3, 1]), int(pos[4, 0]), int(pos[5, 0])]
  pos[3, 1], pos[4, 0], pos[5, 0] = -5, 2**31 - 1, n
  c_order = Order(pos.data_ptr(), order.offsets.data_ptr(), tokens, choices,
                  experts)
  i32, i64 = ctypes.c_int32, ctypes.c_int64
  lib = _native.load_library()
  stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
  new = lambda: torch.full((n + past, dim), HELD, device="cuda")

  def check(got, expected):
    expected = torch.cat([expected, got.new_full((past, dim), HELD)])
    expected[lost] = HELD
    assert torch.equal(got, expected)

  rows = new()
  assert lib.scemb_tokens_to_experts(
      _args(x), i32(0), i64(dim), i64(dim), ctypes.byref(c_order), _args(rows),
      stream) == 0
  check(rows, dense.tokens_to_experts(x, order))

  drows, dw = new(), torch.full((n + past,), HELD, device="cuda")
  assert lib.scemb_tokens_from_experts_grad(
      _args(x), i64(dim), _args(rows_in), i32(0), i64(dim), i64(dim), _args(w),
      i32(0), ctypes.byref(c_order), _args(drows), _args(dw), stream) == 0
  expected, dw_expected = dense.tokens_from_experts_grad(x, rows_in, w, order)
  check(drows, expected)
  dw_expected[3, 1] = dw_expected[4, 0] = dw_expected[5, 0] = 0.0
  assert torch.equal(dw[:n], dw_expected.view(-1)) and (dw[n:] == HELD).all()
