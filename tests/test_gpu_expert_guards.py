"""The C entries of the experts' products write their results and the workspace
they ask for, and nothing beside them, whatever the offsets hold.

Results and workspaces lie in larger buffers filled with a byte that nothing
writes there; the workspace is exactly as large as the size function says.
"""

import ctypes

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore import _native  # pylint: disable=g-import-not-at-top,wrong-import-position
from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

VP, I32, I64, SZ = (ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64,
                    ctypes.c_size_t)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
GUARD, FILL = 1 << 20, 0xa5


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


class _Guarded:
  """`size` bytes between two guards."""

  def __init__(self, size):
    self.size = size
    self.room = torch.full((2 * GUARD + size,), FILL, dtype=torch.uint8,
                           device="cuda")

  def at(self):
    return VP(self.room.data_ptr() + GUARD)

  def inside(self):
    return self.room[GUARD:GUARD + self.size]

  def whole(self):
    return bool((self.room[:GUARD] == FILL).all() and
                (self.room[GUARD + self.size:] == FILL).all())


def _size(name, *args):
  f = getattr(_native.load_library(), name)
  f.restype = SZ
  return f(*args)


def _call(name, *args):
  assert getattr(_native.load_library(), name)(*args) == 0
  torch.cuda.synchronize()


def _stream():
  return VP(torch.cuda.current_stream().cuda_stream)


def _whole(shape, dtype, seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return torch.randint(-3, 4, shape, device="cuda", generator=g).to(dtype)


def _cases(experts, n):
  """Offsets that fit, fall, are negative, overlap, or are past the rows."""
  e = experts + 1
  top = 2**31 - 1
  return [
      [i * n // experts for i in range(e)],
      [n - i * n // experts for i in range(e)],
      [-7 - i for i in range(e)],
      [n + 1 + i for i in range(e)],
      [-2**31] + [top] * experts,
      [(0, n)[i % 2] for i in range(e)],
      [(top, -2**31)[i % 2] for i in range(e)],
      [(n // 2, n // 3, top)[i % 3] for i in range(e)],
      [0] * experts + [top],
  ]


# Rows, experts, inner, outer: small tiles, cut along the sum, middle tiles and
# large ones; whole 16 bytes a row or not.
SHAPES = [(50, 3, 16, 8), (300, 70, 33, 7), (100, 2, 4096, 64),
          (30_001, 9, 100, 131), (16_300, 5, 264, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,experts,inner,outer", SHAPES)
def test_products(n, experts, inner, outer, dtype):
  x, w = _whole((n, inner), dtype, 1), _whole((experts, inner, outer), dtype,
                                              2)
  code, size = I32(CODE[dtype]), x.element_size()
  ws = _Guarded(_size("scemb_expert_matmul_workspace_size", code, I64(n),
                      I64(inner), I64(outer), I32(experts)))
  y = _Guarded(n * outer * size)
  for i, offsets in enumerate(_cases(experts, n)):
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y.inside().zero_()
    _call("scemb_expert_matmul", VP(x.data_ptr()), code, I64(inner), I64(n),
          I64(inner), I64(outer), VP(w.data_ptr()), I64(inner * outer),
          I64(outer), I64(1), VP(off.data_ptr()), I32(experts), y.at(),
          ws.at(), SZ(ws.size), _stream())
    assert y.whole() and ws.whole(), offsets[:4]
    if i == 0:
      order = dense.ExpertOrder(None, None, off)
      assert torch.equal(y.inside().view(dtype).view(n, outer),
                         dense.expert_matmul(x, w, order))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,experts,inner,outer", SHAPES + [
    (20_000, 9, 16, 8), (4000, 64, 264, 520), (4000, 300, 72, 40)])
def test_weights_gradients(n, experts, inner, outer, dtype):
  x, dy = _whole((n, inner), dtype, 1), _whole((n, outer), dtype, 2)
  code, size = I32(CODE[dtype]), x.element_size()
  ws = _Guarded(_size("scemb_expert_matmul_weights_grad_workspace_size", code,
                      I64(n), I64(inner), I64(outer), I32(experts)))
  dw = _Guarded(experts * inner * outer * size)
  for i, offsets in enumerate(_cases(experts, n)):
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    dw.inside().zero_()
    _call("scemb_expert_matmul_weights_grad", VP(x.data_ptr()), I64(inner),
          VP(dy.data_ptr()), I64(outer), code, I64(n), I64(inner), I64(outer),
          VP(off.data_ptr()), I32(experts), dw.at(), ws.at(), SZ(ws.size),
          _stream())
    assert dw.whole() and ws.whole(), offsets[:4]
    if i == 0:
      order = dense.ExpertOrder(None, None, off)
      w = x.new_zeros((experts, inner, outer))
      assert torch.equal(
          dw.inside().view(dtype).view(experts, inner, outer),
          dense.expert_matmul_grad(dy, x, w, order, with_rows=False)[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,experts,inner,outer", [
    (50, 3, 16, 8), (300, 70, 130, 7), (4001, 9, 300, 1000),
    (32_001, 5, 264, 1000)])
def test_8bit_products(n, experts, inner, outer, dtype):
  x, w = _whole((n, inner), dtype, 1), _whole((experts, inner, outer), dtype,
                                              2)
  q = dense.quantize_weights(w)
  ws = _Guarded(_size("scemb_matmul_8bit_workspace_size", I64(n), I64(inner)))
  y = _Guarded(n * outer * x.element_size())
  for i, offsets in enumerate(_cases(experts, n)):
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    # Rows that are not brought to 8 bits leave the workspace as it is: zeros.
    ws.inside().zero_()
    y.inside().zero_()
    _call("scemb_matmul_8bit", VP(x.data_ptr()), I32(CODE[dtype]), I64(inner),
          I64(n), I64(inner), I64(outer), VP(q.codes.data_ptr()),
          VP(q.exponents.data_ptr()), VP(off.data_ptr()), I32(experts), y.at(),
          ws.at(), SZ(ws.size), _stream())
    assert y.whole() and ws.whole(), offsets[:4]
    if i == 0:
      order = dense.ExpertOrder(None, None, off)
      assert torch.equal(y.inside().view(dtype).view(n, outer),
                         dense.matmul_8bit(x, q, order))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(8, 16), (130, 7), (300, 257)])
def test_codes(inner, outer, dtype):
  w = _whole((3, inner, outer), dtype, 1)
  expected = dense.quantize_weights(w)
  codes = _Guarded(expected.codes.numel())
  exponents = _Guarded(expected.exponents.numel() * 4)
  _call("scemb_quantize_weights", VP(w.data_ptr()), I32(CODE[dtype]),
        I64(inner * outer), I64(outer), I64(1), I64(inner), I64(outer), I32(3),
        codes.at(), exponents.at(), _stream())
  assert codes.whole() and exponents.whole()
  assert torch.equal(codes.inside(),
                     expected.codes.view(torch.uint8).reshape(-1))
  assert torch.equal(exponents.inside().view(torch.int32),
                     expected.exponents.reshape(-1))
