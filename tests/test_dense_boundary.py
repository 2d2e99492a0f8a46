"""What the dense operators' C entries refuse before anything is launched, and
what the Python layer does without a GPU (no GPU needed)."""

import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from jax_tpu_embedding.sparsecore import _native  # pylint: disable=g-import-not-at-top,wrong-import-position
from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

F32, BF16 = 0, 1
OK, INVALID, WORKSPACE = 0, 1, 3
VP, I32, I64, F, SZ = (ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64,
                       ctypes.c_float, ctypes.c_size_t)
SOME = 4096  # an address that is not null; nothing reads it


class Order(ctypes.Structure):
  _fields_ = [("positions", VP), ("offsets", VP), ("tokens", I64),
              ("choices", I32), ("num_experts", I32)]


class State(ctypes.Structure):
  _fields_ = [("m", VP), ("v", VP), ("m_scale", VP), ("v_scale", VP),
              ("size", I64), ("bits", I32), ("reserved", I32),
              ("scratch", VP)]


class Options(ctypes.Structure):
  _fields_ = [(n, ctypes.c_double) for n in
              ("learning_rate", "beta_1", "beta_2", "epsilon", "weight_decay",
               "grad_scale")] + [("step", I64), ("learning_rate_ptr", VP),
                                 ("step_ptr", VP), ("grad_scale_ptr", VP)]


def _call(name, *args):
  f = getattr(_native.load_library(), name)
  return f(*args)


def _norm(x=SOME, dtype=F32, rows=4, dim=8, stride=8, wtype=F32, y=SOME):
  return _call("scemb_layer_norm", VP(x), I32(dtype), I64(rows), I64(dim),
               I64(stride), VP(0), VP(0), I32(wtype), F(1e-6), VP(y), VP(0),
               VP(0), VP(0))


@pytest.mark.parametrize("bad", [
    dict(x=0), dict(y=0), dict(dtype=3), dict(dtype=-1), dict(rows=-1),
    dict(dim=0), dict(dim=2**31), dict(stride=-8),
    dict(dtype=F32, wtype=BF16), dict(dtype=BF16, wtype=2)])
def test_layer_norm(bad):
  assert _norm(**bad) == INVALID
  assert _native.load_library().scemb_last_error()
  assert _norm(rows=0) == OK


def test_layer_norm_grad():
  def call(dy=SOME, rows=4, dim=8, weight_grad=SOME, ws=SOME, size=1 << 20,
           dtype=F32):
    return _call("scemb_layer_norm_grad", VP(dy), I64(dim), VP(SOME), I64(dim),
                 I32(dtype), I64(rows), I64(dim), VP(SOME), VP(SOME), VP(0),
                 I32(F32), VP(SOME), VP(weight_grad), VP(0), VP(ws), SZ(size),
                 VP(0))
  assert call(dy=0) == INVALID
  assert call(dim=0) == INVALID
  assert call(dtype=7) == INVALID
  assert call(ws=0) == WORKSPACE
  assert call(size=8) == WORKSPACE
  assert call(rows=0, weight_grad=0) == OK
  size = _native.load_library().scemb_layer_norm_grad_workspace_size
  size.restype = SZ
  assert size(I32(F32), I64(4), I64(0)) == 0
  assert size(I32(9), I64(4), I64(8)) == 0
  assert size(I32(F32), I64(0), I64(8)) > 0


def test_sort_by_expert():
  def call(ids=SOME, width=8, n=100, experts=4, ws=SOME, size=1 << 20,
           offsets=SOME):
    return _call("scemb_sort_by_expert", VP(ids), I32(width), I64(n),
                 I32(experts), VP(SOME), VP(SOME), VP(offsets), VP(ws),
                 SZ(size), VP(0))
  for bad in (dict(ids=0), dict(width=2), dict(n=-1), dict(n=2**31),
              dict(experts=0), dict(experts=1025), dict(offsets=0)):
    assert call(**bad) == INVALID
  assert call(n=100_000, ws=0) == WORKSPACE
  assert call(n=100_000, size=16) == WORKSPACE
  size = _native.load_library().scemb_sort_by_expert_workspace_size
  size.restype = SZ
  assert size(I64(-1), I32(4)) == 0 and size(I64(10), I32(0)) == 0
  # None for one work-group; no choices are no division by zero.
  assert size(I64(100), I32(4)) == 0 and size(I64(0), I32(1019)) == 0
  assert size(I64(100_000), I32(4)) > 0
  for experts in (1020, 1024):
    assert size(I64(0), I32(experts)) > 0


@pytest.mark.parametrize("bad", [
    dict(tokens=-1), dict(choices=0), dict(experts=0), dict(experts=1025),
    dict(tokens=2**30, choices=4), dict(dim=0), dict(dtype=5), dict(x=0),
    dict(positions=0), dict(offsets=0), dict(stride=-1)])
def test_experts(bad):
  def args(x=SOME, dtype=F32, stride=8, dim=8, tokens=4, choices=2, experts=4,
           positions=SOME, offsets=SOME):
    return x, dtype, stride, dim, Order(positions, offsets, tokens, choices,
                                        experts)
  x, dtype, stride, dim, order = args(**bad)
  o = ctypes.byref(order)
  assert _call("scemb_tokens_to_experts", VP(x), I32(dtype), I64(stride),
               I64(dim), o, VP(SOME), VP(0)) == INVALID
  assert _call("scemb_tokens_from_experts", VP(x), I32(dtype), I64(stride),
               I64(dim), VP(0), I32(F32), o, VP(SOME), VP(0)) == INVALID
  assert _call("scemb_tokens_from_experts_grad", VP(x), I64(stride), VP(x),
               I32(dtype), I64(stride), I64(dim), VP(0), I32(F32), o, VP(SOME),
               VP(0), VP(0)) == INVALID
  x, dtype, stride, dim, order = args(tokens=0, x=0)
  assert _call("scemb_tokens_to_experts", VP(0), I32(F32), I64(8), I64(8),
               ctypes.byref(order), VP(0), VP(0)) == OK
  assert _call("scemb_tokens_to_experts", VP(SOME), I32(F32), I64(8), I64(8),
               VP(0), VP(SOME), VP(0)) == INVALID


def _tensors(*rows):
  out = np.zeros(len(rows), dense._TENSOR)  # pylint: disable=protected-access
  for i, r in enumerate(rows):
    for k, v in r.items():
      out[i][k] = v
  return out


def test_adamw():
  one = dict(param=SOME, grad=SOME, numel=300)
  def call(rows=(one,), state=None, options=None, n=None):
    t = _tensors(*rows)
    s = State(**{**dict(m=SOME, v=SOME, size=512, bits=32), **(state or {})})
    o = Options(**{**dict(learning_rate=0.1, beta_1=0.9, beta_2=0.99,
                          epsilon=1e-8, grad_scale=1.0, step=1),
                   **(options or {})})
    return _call("scemb_adamw_update", VP(t.ctypes.data),
                 I32(len(rows) if n is None else n), ctypes.byref(s),
                 ctypes.byref(o), VP(0))
  bad = [
      dict(rows=({**one, "param": 0},)), dict(rows=({**one, "numel": -1},)),
      dict(rows=({**one, "param_type": 2},)),
      dict(rows=({**one, "grad_type": 2},)),
      dict(rows=({**one, "numel": 513},)), dict(rows=(one, one)),
      dict(state=dict(bits=16)), dict(state=dict(size=500)),
      dict(state=dict(size=-256)), dict(state=dict(m=0)),
      dict(state=dict(v=0)), dict(state=dict(bits=8)),
      dict(options=dict(step=0)), dict(n=-1),
      dict(options=dict(step_ptr=SOME)),
      dict(options=dict(learning_rate_ptr=SOME))]
  for b in bad:
    assert call(**b) == INVALID, b
  # Nothing to do: no tensors, none with a gradient, none with values.
  assert call(rows=()) == OK
  assert call(rows=({**one, "grad": 0},)) == OK
  assert call(rows=({**one, "numel": 0},)) == OK
  s = State(m=SOME, v=SOME, size=512, bits=32)
  assert _call("scemb_adamw_moments", ctypes.byref(s), VP(SOME), VP(SOME),
               VP(0)) == INVALID


def test_binding_loads_and_needs_a_gpu():
  calls = _native.dense_binding()
  for name in ("layer_norm", "layer_norm_grad", "sort_by_expert",
               "tokens_to_experts", "tokens_from_experts",
               "tokens_from_experts_grad", "adamw_update", "adamw_moments"):
    assert callable(getattr(calls, name))
  with pytest.raises(ValueError):
    calls.bind([1, 2])
  x = torch.zeros((2, 3))
  assert not calls.wants_grad(x, None)
  assert calls.wants_grad(None, x.requires_grad_())
  with torch.no_grad():
    assert not calls.wants_grad(x)
  if not torch.cuda.is_available():
    with pytest.raises(RuntimeError):
      dense.layer_norm(x)


def test_constants_agree_with_the_header():
  text = open(_native._PKG_ROOT.parent / "include" / "scemb.h").read()  # pylint: disable=protected-access
  assert f"#define SCEMB_ADAMW_BLOCK {dense.ADAMW_BLOCK}\n" in text
  assert f"#define SCEMB_MAX_EXPERTS {dense.MAX_EXPERTS}\n" in text
