"""Products in 8-bit floating point (lib/nn/dense.py) against the definition in
64 bits.

Codes are compared bit for bit: a block's power of two is a whole number of
exponents, and a value divided by it is exact. Products of whole numbers up to 3
are exact throughout. For others the sum of n products of codes is off by at
most n roundings, each of a step (2u, u = 2^-24) of the magnitudes' sum, and the
result's own rounding is half a step of its type. The instructions of 16-bit
results add eight products at a time, each cut to a multiple of 2^(x - 13), 2^x
being the power of two of the largest (256 * 256 + 8 is exact and 256 * 256 + 4
is 256 * 256 there): with the largest itself exact, seven remainders below 2^-13
of it, 7 * 2^-13 of the magnitudes' sum at most. (float32 results are those of
bfloat16 products, which are exact.)
"""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
B = 128


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _order(offsets):
  return dense.ExpertOrder(None, None, torch.tensor(
      offsets, dtype=torch.int32, device="cuda"))


def _values(shape, dtype, seed, whole=False):
  g = torch.Generator(device="cuda").manual_seed(seed)
  if whole:
    return torch.randint(-3, 4, shape, device="cuda", generator=g).to(dtype)
  x = torch.randn(shape, device="cuda", generator=g)
  # Blocks of different sizes, and values of different sizes within them.
  x = x * torch.exp(3 * torch.randn(shape[:-1] + (1,), device="cuda",
                                    generator=g))
  return x.clamp(-6e4, 6e4).to(dtype)


def _exponent(top):
  """The least e >= -126 with top <= 448 * 2^e."""
  if top == 0:
    return -126
  e = math.frexp(top / 448)[1]
  while top <= 448 * 2.0**(e - 1):
    e -= 1
  return max(e, -126)


def _rounded(x, e):
  """x / 2^e in e4m3, as values times 2^e, 64 bits."""
  v = x.double() * 2.0**-e
  step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
  return torch.round(v / step) * step * 2.0**e


def _quantized(x, block):
  """What a matrix's blocks (rows, columns) hold, 64 bits, on the CPU."""
  x = x.double().cpu()
  out = torch.zeros_like(x)
  for i in range(0, x.shape[0], block[0]):
    for j in range(0, x.shape[1], block[1]):
      part = x[i:i + block[0], j:j + block[1]]
      out[i:i + block[0], j:j + block[1]] = _rounded(
          part, _exponent(float(part.abs().max())))
  return out


def _decoded(q, expert=None):
  codes, exponents = q.codes, q.exponents
  if expert is not None:
    codes, exponents = codes[expert], exponents[expert]
  v = codes.float().double().cpu()
  s = torch.exp2(exponents.double().cpu() - 127)
  s = s.repeat_interleave(B, 0).repeat_interleave(B, 1)
  return (v * s[:v.shape[0]])[:, :q.inner].t()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(1, 1), (128, 128), (130, 257),
                                         (300, 60), (127, 129)])
def test_weights(inner, outer, dtype):
  w = _values((inner, outer), dtype, 1)
  q = dense.quantize_weights(w)
  assert q.inner == inner and q.codes.dtype == torch.float8_e4m3fn
  assert q.codes.shape == (outer, -(-inner // B) * B)
  assert not q.codes[:, inner:].float().any()
  assert torch.equal(_decoded(q), _quantized(w, (B, B)))
  # Other memory, the same codes.
  room = torch.full((inner, 2 * outer), float("nan"), dtype=dtype,
                    device="cuda")
  room[:, ::2] = w
  for other in (w.t().contiguous().t(), room[:, ::2]):
    o = dense.quantize_weights(other)
    assert torch.equal(o.codes.view(torch.uint8), q.codes.view(torch.uint8))
    assert torch.equal(o.exponents, q.exponents)


def test_weights_of_experts():
  w = _values((5, 140, 150), torch.bfloat16, 2)
  q = dense.quantize_weights(w)
  for e in range(5):
    assert torch.equal(_decoded(q, e), _quantized(w[e], (B, B)))
    one = dense.quantize_weights(w[e])
    assert torch.equal(one.codes.view(torch.uint8),
                       q.codes[e].view(torch.uint8))


@pytest.mark.parametrize("top", [448.0, 449.0, 447.0, 448 * 2.0**-100,
                                 2.0**-140, 0.0, 3e38, 1.75, 1.7500001])
def test_borders_of_scales(top):
  w = torch.zeros((128, 2), device="cuda")
  w[5, 1] = -top
  w[6, 0] = top / 3
  q = dense.quantize_weights(w)
  assert int(q.exponents[0, 0]) - 127 == _exponent(
      float(torch.tensor(top, dtype=torch.float32)))
  assert torch.equal(_decoded(q), _quantized(w, (B, B)))


def _expected(x, w, offsets):
  """(y, the sum of the magnitudes) of codes, 64 bits."""
  x = _quantized(x, (1, B))
  y = torch.zeros((x.shape[0], w[0].shape[1]), dtype=torch.float64)
  size = torch.zeros_like(y)
  for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
    y[a:b] = x[a:b] @ w[e]
    size[a:b] = x[a:b].abs() @ w[e].abs()
  return y, size


def _check(got, exact, size, inner):
  cut = 7 * 2.0**-13 if got.dtype != torch.float32 else 0.0
  bound = ((2 * U * (inner + 2) + cut) * size +
           torch.finfo(got.dtype).eps / 2 * exact.abs() + 1e-7 * (
               got.dtype == torch.float16))
  got = got.double().cpu()
  near = (got - exact).abs() <= bound
  # float16 is infinite from 65520 on.
  assert (near | (got.isinf() & (exact.abs() > 65000))).all()


SIZES = [(1, 1), (64, 64), (128, 32), (130, 129), (256, 256), (384, 40),
         (1000, 300)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", SIZES)
@pytest.mark.parametrize("rows", [1, 31, 33, 127, 300])
def test_plain_product(rows, inner, outer, dtype):
  for whole in (True, False):
    x, w = _values((rows, inner), dtype, 1, whole), _values(
        (inner, outer), dtype, 2, whole)
    q = dense.quantize_weights(w)
    y = dense.matmul_8bit(x, q)
    assert y.dtype == dtype and y.shape == (rows, outer)
    if whole:
      assert torch.equal(y, (x.double() @ w.double()).to(dtype))
    else:
      _check(y, *_expected(x, [_decoded(q)], [0, rows]), inner)


COUNTS = {
    "single_rows": [1] * 9,
    "some_empty": [0, 5, 0, 33, 0, 1],
    "ragged": [127, 1, 129, 300],
    "many_rows": [700, 0, 513],
    "many_experts": [i % 3 for i in range(1024)],
    "all_dropped": [0, 0],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("inner,outer", [(140, 24), (384, 264)])
def test_rows_of_experts(counts, inner, outer, dtype):
  offsets = [0]
  for c in COUNTS[counts]:
    offsets.append(offsets[-1] + c)
  n, experts = offsets[-1] + 7, len(offsets) - 1
  if experts > 100:
    inner, outer = 36, 40
  for whole in (True, False):
    x = _values((n, inner), dtype, 1, whole)
    w = _values((experts, inner, outer), dtype, 2, whole)
    x[offsets[-1]:] = float("nan")
    q = dense.quantize_weights(w)
    y = dense.matmul_8bit(x, q, _order(offsets))
    assert not y[offsets[-1]:].any()
    x[offsets[-1]:] = 0
    if whole:
      order = _order(offsets)
      assert torch.equal(y, dense.expert_matmul(x, w, order))
    else:
      _check(y, *_expected(x, [_decoded(q, e) for e in range(experts)],
                           offsets), inner)


def test_rows_in_other_memory():
  x, w = _values((50, 140), torch.bfloat16, 1), _values((140, 70),
                                                        torch.bfloat16, 2)
  q = dense.quantize_weights(w)
  y = dense.matmul_8bit(x, q)
  room = torch.full((50, 151), float("nan"), dtype=torch.bfloat16,
                    device="cuda")
  room[:, 3:143] = x
  for other in (room[:, 3:143], x.t().contiguous().t(),
                torch._neg_view(-x)):  # pylint: disable=protected-access
    assert torch.equal(dense.matmul_8bit(other, q), y)
  odd = torch.empty(q.codes.numel() + 1, dtype=torch.uint8, device="cuda")
  odd[1:] = q.codes.view(torch.uint8).reshape(-1)
  moved = q._replace(codes=odd[1:].view(torch.float8_e4m3fn).view(
      q.codes.shape))
  assert torch.equal(dense.matmul_8bit(x, moved), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(bad, dtype):
  x, w = _values((200, 300), dtype, 1, True), _values((300, 200), dtype, 2,
                                                      True)
  y = dense.matmul_8bit(x, dense.quantize_weights(w))
  x[7, 299] = bad
  got = dense.matmul_8bit(x, dense.quantize_weights(w))
  assert got[7].isnan().all()
  keep = torch.arange(200, device="cuda") != 7
  assert torch.equal(got[keep], y[keep])
  # A block of weights: the columns that share it.
  w[0, 130] = bad
  got = dense.matmul_8bit(x, dense.quantize_weights(w))
  assert got[:, 128:].isnan().all()
  assert torch.equal(got[keep][:, :128], y[keep][:, :128])


def test_scales_of_any_size():
  """Rows and weights far from one: the powers of two multiply exactly."""
  x, w = _values((40, 256), torch.float32, 1, True), _values(
      (256, 64), torch.float32, 2, True)
  y = (x.double() @ w.double()).float()
  for a, b in ((2.0**100, 2.0**-100), (2.0**-110, 2.0**100), (2.0**60, 1.0)):
    got = dense.matmul_8bit(x * a, dense.quantize_weights(w * b))
    assert torch.equal(got, y * (a * b))


def test_no_rows():
  q = dense.quantize_weights(torch.ones((8, 16), device="cuda"))
  assert dense.matmul_8bit(torch.empty((0, 8), device="cuda"),
                           q).shape == (0, 16)


def test_captured_and_replayed():
  x, w = _values((300, 260), torch.bfloat16, 1), _values((3, 260, 130),
                                                         torch.bfloat16, 2)
  q, order = dense.quantize_weights(w), _order([0, 100, 120, 290])
  expected = dense.matmul_8bit(x, q, order)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    y = dense.matmul_8bit(x, q, order)
  for _ in range(3):
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, expected)
    assert torch.equal(dense.matmul_8bit(x, q, order), expected)


def test_refusals():
  x, w = torch.ones((6, 8), device="cuda"), torch.ones((8, 4), device="cuda")
  q = dense.quantize_weights(w)
  many = dense.quantize_weights(torch.ones((2, 8, 4), device="cuda"))
  order = _order([0, 3, 6])
  dense.matmul_8bit(x, many, order)
  for bad in (
      lambda: dense.quantize_weights(w[0]),
      lambda: dense.quantize_weights(w[:0]),
      lambda: dense.quantize_weights(w.double()),
      lambda: dense.quantize_weights(w.cpu()),
      lambda: dense.quantize_weights([1.0]),
      lambda: dense.quantize_weights(w[None, None]),
      lambda: dense.quantize_weights(w[:1, :1].expand(1025, 8, 4)),
      lambda: dense.quantize_weights(w[:1].expand((1 << 22) + 1, 4)),
      lambda: dense.matmul_8bit(x[:, :7], q),
      lambda: dense.matmul_8bit(x[0], q),
      lambda: dense.matmul_8bit(x.double(), q),
      lambda: dense.matmul_8bit(x.cpu(), q),
      lambda: dense.matmul_8bit(x, q, order),
      lambda: dense.matmul_8bit(x, many),
      lambda: dense.matmul_8bit(x, many, _order([0, 6])),
      lambda: dense.matmul_8bit(x, q._replace(codes=q.codes.float())),
      lambda: dense.matmul_8bit(x, q._replace(codes=q.codes[:, :64])),
      lambda: dense.matmul_8bit(x, q._replace(exponents=q.exponents[:, :0])),
      lambda: dense.matmul_8bit(x, q._replace(exponents=q.exponents.long())),
      lambda: dense.matmul_8bit(x.clone().requires_grad_(), q)):
    with pytest.raises(ValueError):
      bad()
  with torch.no_grad():
    dense.matmul_8bit(x.clone().requires_grad_(), q)
