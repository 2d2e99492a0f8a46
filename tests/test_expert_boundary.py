"""What the C entries of the experts' products, the 8-bit products and the
gradients' norm refuse before anything is launched (no GPU needed)."""

import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

from jax_tpu_embedding.sparsecore import _native  # pylint: disable=g-import-not-at-top,wrong-import-position
from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

F32 = 0
OK, INVALID, WORKSPACE = 0, 1, 3
VP, I32, I64, SZ, D = (ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64,
                       ctypes.c_size_t, ctypes.c_double)
SOME = 4096  # an address that is not null; nothing reads it


class Gradient(ctypes.Structure):
  _fields_ = [("data", VP), ("numel", I64), ("type", I32), ("reserved", I32)]


def _call(name, *args):
  return getattr(_native.load_library(), name)(*args)


def _size(name, *args):
  f = getattr(_native.load_library(), name)
  f.restype = SZ
  return f(*args)


SIZES = [dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=2**31 - 1),
         dict(inner=0), dict(inner=2**31), dict(outer=0), dict(outer=2**31),
         dict(experts=0), dict(experts=1025)]


def _product(x=SOME, type=F32, stride=8, rows=4, inner=8, outer=6, w=SOME,  # pylint: disable=redefined-builtin
             se=48, si=6, so=1, offsets=SOME, experts=2, y=SOME, ws=0, size=0):
  return _call("scemb_expert_matmul", VP(x), I32(type), I64(stride), I64(rows),
               I64(inner), I64(outer), VP(w), I64(se), I64(si), I64(so),
               VP(offsets), I32(experts), VP(y), VP(ws), SZ(size), VP(0))


@pytest.mark.parametrize("bad", SIZES + [
    dict(x=0), dict(w=0), dict(offsets=0), dict(y=0), dict(stride=-1),
    dict(se=-1), dict(si=-6), dict(so=2), dict(si=6, so=0)])
def test_expert_matmul(bad):
  assert _product(**bad) == INVALID
  assert _native.load_library().scemb_last_error()
  assert _product(rows=0, x=0, y=0) == OK


def test_expert_matmul_workspace():
  name = "scemb_expert_matmul_workspace_size"
  size = lambda rows, inner, outer, experts: _size(
      name, I32(F32), I64(rows), I64(inner), I64(outer), I32(experts))
  # A few rows and a long sum are cut along it: the parts' sums.
  need = size(100, 4096, 64, 1)
  assert need > 0 and need % (100 * 64 * 4) == 0
  for args in ((100, 64, 64, 1), (100_000, 4096, 4096, 1), (0, 4096, 64, 1),
               (100, 0, 64, 1), (128, 4096, 4096, 64)):
    assert size(*args) == 0
  long = dict(rows=100, inner=4096, stride=4096, outer=64, si=64, se=4096 * 64,
              experts=1)
  assert _product(**long) == WORKSPACE
  assert _product(**long, ws=SOME, size=need - 1) == WORKSPACE


def _weights_grad(x=SOME, dy=SOME, type=F32, rows=100_000, inner=8, outer=6,  # pylint: disable=redefined-builtin
                  offsets=SOME, experts=2, dw=SOME, ws=SOME, size=1 << 28):
  return _call("scemb_expert_matmul_weights_grad", VP(x), I64(inner), VP(dy),
               I64(outer), I32(type), I64(rows), I64(inner), I64(outer),
               VP(offsets), I32(experts), VP(dw), VP(ws), SZ(size), VP(0))


@pytest.mark.parametrize("bad", SIZES + [
    dict(x=0), dict(dy=0), dict(offsets=0), dict(dw=0)])
def test_weights_grad(bad):
  assert _weights_grad(**bad) == INVALID


def test_weights_grad_workspace():
  name = "scemb_expert_matmul_weights_grad_workspace_size"
  size = lambda rows, inner, outer, experts: _size(
      name, I32(F32), I64(rows), I64(inner), I64(outer), I32(experts))
  assert size(100_000, 8, 6, 2) > 0
  assert _weights_grad(ws=0) == WORKSPACE
  assert _weights_grad(size=16) == WORKSPACE
  # None where tiles are many, rows few or the call is refused; sums of pieces
  # are 128 MB at most.
  for args in ((100_000, 8192, 8192, 64), (10, 8, 6, 2), (10, 0, 6, 2),
               (2**30, 2**30, 2**30, 1024)):
    assert size(*args) == 0
  for args in ((100_000, 100, 403, 61), (2**30, 8, 8, 1), (60_000, 512, 512, 9),
               (2**31 - 2**17, 3, 3, 300)):
    assert 0 < size(*args) <= 128 << 20


def _quantize(w=SOME, type=F32, se=48, si=6, so=1, inner=8, outer=6, experts=2,  # pylint: disable=redefined-builtin
              codes=SOME, exponents=SOME):
  return _call("scemb_quantize_weights", VP(w), I32(type), I64(se), I64(si),
               I64(so), I64(inner), I64(outer), I32(experts), VP(codes),
               VP(exponents), VP(0))


@pytest.mark.parametrize("bad", [
    dict(w=0), dict(codes=0), dict(exponents=0), dict(type=3), dict(se=-1),
    dict(so=2), dict(inner=0), dict(inner=2**22 + 1), dict(outer=0),
    dict(experts=0), dict(experts=1025)])
def test_quantize_weights(bad):
  assert _quantize(**bad) == INVALID


def _matmul_8(x=SOME, type=F32, stride=8, rows=4, inner=8, outer=6, codes=SOME,  # pylint: disable=redefined-builtin
              exponents=SOME, offsets=SOME, experts=2, y=SOME, ws=SOME,
              size=1 << 20):
  return _call("scemb_matmul_8bit", VP(x), I32(type), I64(stride), I64(rows),
               I64(inner), I64(outer), VP(codes), VP(exponents), VP(offsets),
               I32(experts), VP(y), VP(ws), SZ(size), VP(0))


@pytest.mark.parametrize("bad", [
    dict(x=0), dict(codes=0), dict(exponents=0), dict(y=0), dict(type=3),
    dict(stride=-1), dict(rows=-1), dict(inner=0), dict(inner=2**22 + 1),
    dict(outer=0), dict(experts=0), dict(experts=1025), dict(offsets=0),
    dict(codes=SOME + 8)])
def test_matmul_8bit(bad):
  assert _matmul_8(**bad) == INVALID
  assert _matmul_8(rows=0, x=0) == OK
  for small in (dict(ws=0), dict(size=16), dict(ws=SOME + 4)):
    assert _matmul_8(**small) == WORKSPACE
  assert _size("scemb_matmul_8bit_workspace_size", I64(-1), I64(8)) == 0


def _norm(entry, rows=((SOME, 10, 0),), n=None, limit=1.0, norm=SOME, ws=SOME,
          size=1 << 20):
  g = (Gradient * max(len(rows), 1))(*[Gradient(*r, 0) for r in rows])
  args = [ctypes.byref(g), I32(len(rows) if n is None else n), D(limit),
          VP(norm)]
  if entry == "scemb_gradient_norm":
    args.append(VP(0))
  return _call(entry, *args, VP(ws), SZ(size), VP(0))


@pytest.mark.parametrize("entry", ["scemb_gradient_norm",
                                   "scemb_clip_gradients"])
def test_gradient_norm(entry):
  for bad in (dict(rows=((0, 10, 0),)), dict(rows=((SOME, -1, 0),)),
              dict(rows=((SOME, 10, 3),)), dict(rows=((SOME, 10, -1),)),
              dict(rows=((SOME, 2**60 + 1, 0),)), dict(n=-1), dict(limit=-1.0),
              dict(limit=math.nan), dict(norm=0)):
    assert _norm(entry, **bad) == INVALID, bad
  for small in (dict(ws=0), dict(size=16)):
    assert _norm(entry, **small) == WORKSPACE


def test_constants_agree_with_the_header():
  text = open(_native._PKG_ROOT.parent / "include" / "scemb.h").read()  # pylint: disable=protected-access
  assert f"#define SCEMB_BLOCK_8BIT {dense.BLOCK_8BIT}\n" in text


def test_binding_has_the_calls_and_needs_a_gpu():
  calls = _native.dense_binding()
  for name in ("expert_matmul", "expert_matmul_grad", "quantize_weights",
               "matmul_8bit", "gradient_norm", "clip_gradients"):
    assert callable(getattr(calls, name))
  if not torch.cuda.is_available():
    for call in (lambda: dense.quantize_weights(torch.zeros(2, 2)),
                 lambda: dense.gradient_norm([torch.zeros(2)])):
      with pytest.raises(RuntimeError):
        call()
