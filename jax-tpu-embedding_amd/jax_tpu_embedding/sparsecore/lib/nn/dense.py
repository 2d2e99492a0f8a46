"""The dense operators of a ranking model that trains beside its tables.

No counterpart in the reference, whose users take these from their framework's
compiler. Three families, each a hand-written gfx950 kernel behind the C ABI:

  layer_norm, layer_norm_grad
      layer norm of the activations that the lookups return, and its
      gradients, the weight's and the bias's included;
  sort_by_expert, tokens_to_experts, tokens_from_experts (and their _grad)
      a mixture of experts' tokens in the order of their experts and back,
      with the router's weights applied;
  init_adamw_state, adamw_update, adamw_moments
      AdamW over all dense weights in one or a few launches, with moments in
      float32 or in 8 bits.

Arrays are torch tensors on the current GPU, work is enqueued on the current
stream and nothing waits for it. layer_norm, tokens_to_experts and
tokens_from_experts take part in torch's autograd; the _grad functions are the
same gradients for callers that keep their own tape, as
embedding.tpu_sparse_dense_matmul_grad's are.
"""

from __future__ import annotations

from typing import NamedTuple

import numpy as np

from jax_tpu_embedding.sparsecore import _native

ADAMW_BLOCK = _native.ADAMW_BLOCK
MAX_EXPERTS = _native.MAX_EXPERTS

_type_codes = None


def _types():
  """torch dtype -> type code of the C ABI."""
  global _type_codes
  if _type_codes is None:
    t = _native.torch()
    _type_codes = {t.float32: _native.TYPE_F32, t.bfloat16: _native.TYPE_BF16,
                   t.float16: _native.TYPE_F16}
  return _type_codes


def _check_tensor(x, name: str, dtypes) -> None:
  t = _native.require_gpu()
  if not isinstance(x, t.Tensor):
    raise ValueError(f"{name} must be a torch tensor, got {type(x).__name__}")
  if not x.is_cuda or x.get_device() != t.cuda.current_device():
    raise ValueError(f"{name} must be on the current GPU, it is on {x.device}")
  if x.dtype not in dtypes:
    raise ValueError(f"{name} must be one of "
                     f"{', '.join(str(d) for d in dtypes)}, got {x.dtype}")


def _rows_of(x, dim: int):
  """x as a matrix of rows of `dim` neighbouring values, and how many values
  apart the rows are (a copy where x's strides allow no such view)."""
  if x.dim() != 2:
    x = x.reshape(-1, dim)
  if x.stride(1) != 1 and dim != 1:
    x = x.contiguous()
  return x, x.stride(0)


def _wants_grad(*tensors) -> bool:
  return _native.torch().is_grad_enabled() and any(
      x is not None and x.requires_grad for x in tensors)


_functions = {}


def _function(name: str):
  """The autograd functions, made on first use: torch is imported late."""
  if not _functions:
    t = _native.torch()
    once = t.autograd.function.once_differentiable

    class LayerNorm(t.autograd.Function):

      @staticmethod
      def forward(ctx, x, weight, bias, epsilon):
        y, mean, rstd = _layer_norm(x, weight, bias, epsilon, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias = None if bias is None else bias.dtype
        ctx.mark_non_differentiable(mean, rstd)
        return y, mean, rstd

      @staticmethod
      @once
      def backward(ctx, y_grad, *_):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _layer_norm_grad(
            y_grad, x, mean, rstd, weight, need[1] and weight is not None,
            ctx.bias if need[2] else None)
        return dx if need[0] else None, dw, db, None

    class ToExperts(t.autograd.Function):

      @staticmethod
      def forward(ctx, x, positions, offsets):
        ctx.save_for_backward(positions, offsets)
        return _to_experts(x, positions, offsets)

      @staticmethod
      @once
      def backward(ctx, rows_grad):
        return _from_experts(rows_grad, None, *ctx.saved_tensors), None, None

    class FromExperts(t.autograd.Function):

      @staticmethod
      def forward(ctx, rows, weights, positions, offsets):
        ctx.save_for_backward(rows, weights, positions, offsets)
        return _from_experts(rows, weights, positions, offsets)

      @staticmethod
      @once
      def backward(ctx, y_grad):
        rows, weights, positions, offsets = ctx.saved_tensors
        need = ctx.needs_input_grad
        drows, dw = _from_experts_grad(y_grad, rows, weights, positions,
                                       offsets)
        return (drows if need[0] else None, dw if need[1] else None, None,
                None)

    _functions.update(norm=LayerNorm, to=ToExperts, back=FromExperts)
  return _functions[name]


# ---------------------------------------------------------------------------
# Layer norm.
# ---------------------------------------------------------------------------


def _check_affine(p, name: str, x, dim: int) -> None:
  _check_tensor(p, name, dict.fromkeys((_native.torch().float32, x.dtype)))
  if tuple(p.shape) != (dim,):
    raise ValueError(f"{name} must have shape ({dim},), got {tuple(p.shape)}")


def _check_norm(x, weight, bias) -> int:
  _check_tensor(x, "x", _types())
  if x.dim() < 1 or x.shape[-1] < 1:
    raise ValueError("x must have a last dimension of at least 1, got shape "
                     f"{tuple(x.shape)}")
  dim = x.shape[-1]
  if weight is not None:
    _check_affine(weight, "weight", x, dim)
  if bias is not None:
    _check_affine(bias, "bias", x, dim)
    if weight is not None and weight.dtype != bias.dtype:
      raise ValueError("weight and bias must be of one type, got "
                       f"{weight.dtype} and {bias.dtype}")
  return dim


def _layer_norm(x, weight, bias, epsilon, stats):
  t = _native.torch()
  dim = x.shape[-1]
  y = t.empty(x.shape, dtype=x.dtype, device=x.device)
  rows, stride = _rows_of(x, dim)
  n = rows.shape[0]
  mean = rstd = None
  if stats:
    mean = t.empty(x.shape[:-1], dtype=t.float32, device=x.device)
    rstd = t.empty_like(mean)
  codes = _types()
  weight = None if weight is None else weight.contiguous()
  bias = None if bias is None else bias.contiguous()
  affine = weight if weight is not None else bias
  _native.layer_norm(
      rows, codes[x.dtype], n, dim, stride, weight, bias,
      _native.TYPE_F32 if affine is None else codes[affine.dtype], epsilon, y,
      mean, rstd)
  return y, mean, rstd


def layer_norm(x, weight=None, bias=None, *, epsilon: float = 1e-6,
               return_stats: bool = False):
  """Layer norm of x over its last dimension, of x's type.

  x: float32, bfloat16 or float16, [..., dim]; any strides (rows that are not
    contiguous in the last dimension are copied first).
  weight, bias: [dim], float32 or x's type, the same for both; None: one, zero.
  epsilon: added to the variance.
  return_stats: also return the float32 mean and reciprocal deviation of every
    row ([...]), which layer_norm_grad takes.

  Statistics and products are float32; the result is rounded once. A row that
  holds an infinity or a NaN gives a row of NaN.
  """
  _check_norm(x, weight, bias)
  epsilon = float(epsilon)
  if not epsilon >= 0:
    raise ValueError(f"epsilon must not be negative, got {epsilon}")
  if _wants_grad(x, weight, bias):
    out = _function("norm").apply(x, weight, bias, epsilon)
    return out if return_stats else out[0]
  out = _layer_norm(x, weight, bias, epsilon, return_stats)
  return out if return_stats else out[0]


def _layer_norm_grad(y_grad, x, mean, rstd, weight, want_weight, bias_dtype):
  t = _native.torch()
  dim = x.shape[-1]
  codes = _types()
  dx = t.empty(x.shape, dtype=x.dtype, device=x.device)
  rows, stride = _rows_of(x, dim)
  dy, dy_stride = _rows_of(y_grad, dim)
  new = lambda dtype: t.empty(dim, dtype=dtype, device=x.device)
  dw = new(weight.dtype) if want_weight else None
  db = None if bias_dtype is None else new(bias_dtype)
  affine = weight.dtype if weight is not None else bias_dtype
  _native.layer_norm_grad(
      dy, dy_stride, rows, stride, codes[x.dtype], rows.shape[0], dim,
      mean.contiguous(), rstd.contiguous(),
      None if weight is None else weight.contiguous(),
      _native.TYPE_F32 if affine is None else codes[affine], dx, dw, db)
  return dx, dw, db


def layer_norm_grad(y_grad, x, mean, rstd, weight=None, *,
                    with_bias: bool = True):
  """Gradients of layer_norm: (of x, of weight, of bias).

  y_grad: the gradient of its result, of x's shape and type.
  x, weight: what layer_norm was given; mean, rstd: what it returned.
  with_bias: whether to compute the bias's gradient.

  x's gradient is of x's type. The weight's (None without a weight) and the
  bias's are of the weight's type (float32 without one), summed over the rows
  in float32 in an order that the shapes decide.
  """
  t = _native.require_gpu()
  dim = _check_norm(x, weight, None)
  _check_tensor(y_grad, "y_grad", (x.dtype,))
  if y_grad.shape != x.shape:
    raise ValueError(f"y_grad must have x's shape {tuple(x.shape)}, got "
                     f"{tuple(y_grad.shape)}")
  for s, name in ((mean, "mean"), (rstd, "rstd")):
    _check_tensor(s, name, (t.float32,))
    if s.numel() * dim != x.numel():
      raise ValueError(f"{name} must have a value for each row of x, got shape "
                       f"{tuple(s.shape)}")
  bias = None
  if with_bias:
    bias = t.float32 if weight is None else weight.dtype
  return _layer_norm_grad(y_grad, x, mean, rstd, weight, weight is not None,
                          bias)


# ---------------------------------------------------------------------------
# Tokens and experts.
# ---------------------------------------------------------------------------


class ExpertOrder(NamedTuple):
  """The order of tokens' choices by expert, int32 tensors on the GPU.

  positions: of the shape of the ids: the row of each choice among all,
    expert by expert, dropped choices at the end.
  sources: [choices in all]: the choice (token * choices per token + k) of
    each row.
  offsets: [num_experts + 1]: the first row of each expert; the last is the
    number of choices that are not dropped.
  """

  positions: object
  sources: object
  offsets: object


def sort_by_expert(expert_ids, num_experts: int) -> ExpertOrder:
  """Orders every token's choices of experts by expert.

  expert_ids: int32 or int64, [tokens, choices] or [tokens] (one choice each).
    Ids outside [0, num_experts) are dropped choices (padded samples, an
    expert over its capacity).
  num_experts: 1 to MAX_EXPERTS.

  Choices of one expert keep their order.
  """
  t = _native.require_gpu()
  _check_tensor(expert_ids, "expert_ids", (t.int32, t.int64))
  if expert_ids.dim() not in (1, 2):
    raise ValueError("expert_ids must have shape (tokens, choices) or "
                     f"(tokens,), got {tuple(expert_ids.shape)}")
  num_experts = int(num_experts)
  if not 1 <= num_experts <= MAX_EXPERTS:
    raise ValueError(f"num_experts must be within [1, {MAX_EXPERTS}], got "
                     f"{num_experts}")
  n = expert_ids.numel()
  if n > 2**31 - 1:
    raise ValueError(f"at most 2^31 - 1 choices can be ordered, got {n}")
  new = lambda shape: t.empty(shape, dtype=t.int32, device=expert_ids.device)
  order = ExpertOrder(new(expert_ids.shape), new(n), new(num_experts + 1))
  _native.sort_by_expert(expert_ids.contiguous(), expert_ids.element_size(),
                         num_experts, *order)
  return order


def _order_struct(positions, offsets) -> _native.ExpertOrder:
  return _native.ExpertOrder(
      positions.data_ptr(), offsets.data_ptr(), positions.shape[0],
      1 if positions.dim() == 1 else positions.shape[1],
      offsets.shape[0] - 1)


def _check_order(order):
  """(positions, offsets, tokens) of an ExpertOrder."""
  t = _native.require_gpu()
  positions, offsets = order.positions, order.offsets
  _check_tensor(positions, "order.positions", (t.int32,))
  _check_tensor(offsets, "order.offsets", (t.int32,))
  if positions.dim() not in (1, 2) or (positions.dim() == 2 and
                                       positions.shape[1] < 1):
    raise ValueError("order.positions must have shape (tokens, choices) or "
                     f"(tokens,), got {tuple(positions.shape)}")
  if offsets.dim() != 1 or not 2 <= offsets.shape[0] <= MAX_EXPERTS + 1:
    raise ValueError("order.offsets must have shape (num_experts + 1,), got "
                     f"{tuple(offsets.shape)}")
  return positions.contiguous(), offsets.contiguous(), positions.shape[0]


def _check_rows(x, name: str, n: int, dtypes) -> None:
  _check_tensor(x, name, dtypes)
  if x.dim() != 2 or x.shape[0] != n or x.shape[1] < 1:
    raise ValueError(f"{name} must have shape ({n}, dim), got "
                     f"{tuple(x.shape)}")


def _check_weights(weights, positions, rows) -> None:
  if weights is None:
    return
  _check_tensor(weights, "weights",
                dict.fromkeys((_native.torch().float32, rows.dtype)))
  if weights.shape != positions.shape:
    raise ValueError("weights must have the shape of the ids, "
                     f"{tuple(positions.shape)}, got {tuple(weights.shape)}")


def _weights_type(weights) -> int:
  return _native.TYPE_F32 if weights is None else _types()[weights.dtype]


def _to_experts(x, positions, offsets):
  t = _native.torch()
  dim = x.shape[1]
  x, stride = _rows_of(x, dim)
  rows = t.empty((positions.numel(), dim), dtype=x.dtype, device=x.device)
  _native.tokens_to_experts(x, _types()[x.dtype], stride, dim,
                            _order_struct(positions, offsets), rows)
  return rows


def _from_experts(rows, weights, positions, offsets):
  t = _native.torch()
  dim = rows.shape[1]
  rows, stride = _rows_of(rows, dim)
  y = t.empty((positions.shape[0], dim), dtype=rows.dtype, device=rows.device)
  _native.tokens_from_experts(
      rows, _types()[rows.dtype], stride, dim,
      None if weights is None else weights.contiguous(),
      _weights_type(weights), _order_struct(positions, offsets), y)
  return y


def _from_experts_grad(y_grad, rows, weights, positions, offsets):
  t = _native.torch()
  dim = rows.shape[1]
  dy, dy_stride = _rows_of(y_grad, dim)
  src, stride = _rows_of(rows, dim)
  drows = t.empty(rows.shape, dtype=rows.dtype, device=rows.device)
  dweights = None
  if weights is not None:
    dweights = t.empty(weights.shape, dtype=weights.dtype,
                       device=weights.device)
  _native.tokens_from_experts_grad(
      dy, dy_stride, src, _types()[rows.dtype], stride, dim,
      None if weights is None else weights.contiguous(),
      _weights_type(weights), _order_struct(positions, offsets), drows,
      dweights)
  return drows, dweights


def tokens_to_experts(x, order: ExpertOrder):
  """The tokens' rows in the order of their experts, [choices in all, dim]:
  row order.positions[t, k] is x[t]; rows of dropped choices are zero.

  x: [tokens, dim], float32, bfloat16 or float16.
  """
  positions, offsets, tokens = _check_order(order)
  _check_rows(x, "x", tokens, _types())
  if _wants_grad(x):
    return _function("to").apply(x, positions, offsets)
  return _to_experts(x, positions, offsets)


def tokens_to_experts_grad(rows_grad, order: ExpertOrder):
  """The gradient of tokens_to_experts's x: the sum of the gradients of its
  choices' rows, in float32, rounded once. Rows of dropped choices are not
  read."""
  positions, offsets, _ = _check_order(order)
  _check_rows(rows_grad, "rows_grad", positions.numel(), _types())
  return _from_experts(rows_grad, None, positions, offsets)


def tokens_from_experts(rows, weights, order: ExpertOrder):
  """The experts' rows back at their tokens, [tokens, dim]: the sum over the
  token's choices of weight * row, in float32, rounded once.

  rows: [choices in all, dim]; rows of dropped choices are not read and add
    nothing (a token without choices gets zeros).
  weights: of the ids' shape, float32 or rows' type; None: one.
  """
  positions, offsets, _ = _check_order(order)
  _check_rows(rows, "rows", positions.numel(), _types())
  _check_weights(weights, positions, rows)
  if _wants_grad(rows, weights):
    return _function("back").apply(rows, weights, positions, offsets)
  return _from_experts(rows, weights, positions, offsets)


def tokens_from_experts_grad(y_grad, rows, weights, order: ExpertOrder):
  """Gradients of tokens_from_experts: (of rows, of weights).

  Rows of dropped choices get zeros, and so do their weights. The second is
  None without weights.
  """
  positions, offsets, tokens = _check_order(order)
  _check_rows(rows, "rows", positions.numel(), _types())
  _check_weights(weights, positions, rows)
  _check_tensor(y_grad, "y_grad", (rows.dtype,))
  if tuple(y_grad.shape) != (tokens, rows.shape[1]):
    raise ValueError(f"y_grad must have shape ({tokens}, {rows.shape[1]}), "
                     f"got {tuple(y_grad.shape)}")
  return _from_experts_grad(y_grad, rows, weights, positions, offsets)


# ---------------------------------------------------------------------------
# AdamW.
# ---------------------------------------------------------------------------


class AdamWState:
  """The moments of a list of weights, and the steps taken.

  m, v: the moments of all weights in one tensor each, weight i's from
    first[i] on, first[i] being a multiple of ADAMW_BLOCK. float32, or int8 and
    uint8 with 8 bits, whose values adamw_moments returns.
  m_scale, v_scale: with 8 bits, a float32 for each ADAMW_BLOCK values; else
    None.
  step: updates made so far.
  bits: 8 or 32.

  A checkpoint keeps these tensors and the step; a state made for the same
  weights takes them back with copy_().
  """

  def __init__(self, sizes, decay, bits: int, device):
    t = _native.torch()
    padded = [-(-n // ADAMW_BLOCK) * ADAMW_BLOCK for n in sizes]
    self.first = [0] * len(sizes)
    total = 0
    for i, n in enumerate(padded):
      self.first[i] = total
      total += n
    self.bits = bits
    self.step = 0
    new = lambda n, dtype: t.zeros(n, dtype=dtype, device=device)
    if bits == 8:
      self.m, self.v = new(total, t.int8), new(total, t.uint8)
      self.m_scale = new(total // ADAMW_BLOCK, t.float32)
      self.v_scale = new(total // ADAMW_BLOCK, t.float32)
    else:
      self.m, self.v = new(total, t.float32), new(total, t.float32)
      self.m_scale = self.v_scale = None
    self._table = np.zeros(len(sizes), _native.ADAMW_TENSOR)
    self._table["numel"] = sizes
    self._table["decay"] = decay

  def as_struct(self) -> _native.AdamWState:
    return _native.AdamWState(
        _native.ptr(self.m), _native.ptr(self.v), _native.ptr(self.m_scale),
        _native.ptr(self.v_scale), self.m.numel(), self.bits, 0)


def _adamw_types():
  t = _native.torch()
  return (t.float32, t.bfloat16)


def _check_params(params) -> None:
  types = _adamw_types()
  for i, p in enumerate(params):
    _check_tensor(p, f"params[{i}]", types)
    if not p.is_contiguous():
      raise ValueError(f"params[{i}] must be contiguous")


def init_adamw_state(params, *, state_bits: int = 32,
                     decay=None) -> AdamWState:
  """The state of AdamW before its first step.

  params: a sequence of float32 or bfloat16 tensors, contiguous, of any sizes.
  state_bits: 32 (float32 moments) or 8 (blocks of ADAMW_BLOCK values with a
    scale each: 2.03 bytes a value for both moments instead of 8).
  decay: for each weight whether weight decay applies (None: to all).
  """
  if state_bits not in (8, 32):
    raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
  params = list(params)
  decay = [True] * len(params) if decay is None else [bool(d) for d in decay]
  if len(decay) != len(params):
    raise ValueError(f"decay has {len(decay)} entries for {len(params)} "
                     "params")
  _check_params(params)
  return AdamWState([p.numel() for p in params], decay, state_bits,
                    _native.device())


def _device_scalar(x, dtype):
  """(tensor to keep, address) of a value on the GPU, (None, None) of one on
  the host."""
  t = _native.torch()
  if isinstance(x, t.Tensor) and x.is_cuda:
    if x.numel() != 1:
      raise ValueError("a hyperparameter on the GPU must be one value, got "
                       f"shape {tuple(x.shape)}")
    x = x.to(device=_native.device(), dtype=dtype)
    return x, x.data_ptr()
  return None, None


def adamw_update(params, grads, state: AdamWState, *, learning_rate,
                 beta_1: float = 0.9, beta_2: float = 0.999,
                 epsilon: float = 1e-8, weight_decay: float = 0.01,
                 grad_scale=None, copies=None, step=None):
  """One step of AdamW on all params, in place; returns params.

  With g = grad * grad_scale, t the step, every value of every weight:
    m = beta_1 * m + (1 - beta_1) * g
    v = beta_2 * v + (1 - beta_2) * g * g
    p = p * (1 - learning_rate * weight_decay) - learning_rate
        / (1 - beta_1^t) * m / (sqrt(v) / sqrt(1 - beta_2^t) + epsilon)
  in float32, rounded once to the weight's type. With 8 bits, m and v are
  rounded to their codes after they were used.

  params: the weights that the state was made for (sizes and order).
  grads: a gradient of each, of its shape, float32 or bfloat16; None leaves
    that weight and its moments as they are.
  learning_rate, grad_scale: floats, or single values on the GPU (a schedule's
    or a clipping factor that nobody waits for).
  copies: None, or a bfloat16 tensor of each weight's shape (or None) that gets
    the rounded weight: the working copies of float32 weights.
  step: None (state.step + 1), an int, or a single int64 on the GPU, which a
    captured graph advances itself. The first step is 1.
  """
  t = _native.require_gpu()
  params, grads = list(params), list(grads)
  n = len(params)
  table = state._table  # pylint: disable=protected-access
  if len(table) != n or len(grads) != n:
    raise ValueError(f"{n} params and {len(grads)} grads for a state of "
                     f"{len(table)}")
  copies = [None] * n if copies is None else list(copies)
  if len(copies) != n:
    raise ValueError(f"{len(copies)} copies for {n} params")
  if not (0 <= beta_1 < 1 and 0 <= beta_2 < 1 and epsilon >= 0):
    raise ValueError("beta_1 and beta_2 must be within [0, 1) and epsilon not "
                     f"negative, got {beta_1}, {beta_2} and {epsilon}")
  _check_params(params)
  _check_tensor(state.m, "state.m", (state.m.dtype,))
  types, codes = _adamw_types(), _types()
  keep = []
  rows = []
  for i, (p, g, c) in enumerate(zip(params, grads, copies)):
    ga = ca = gt = 0
    if g is not None:
      _check_tensor(g, f"grads[{i}]", types)
      if g.shape != p.shape:
        raise ValueError(f"grads[{i}] must have the shape {tuple(p.shape)} of "
                         f"its weight, got {tuple(g.shape)}")
      if not g.is_contiguous():
        g = g.contiguous()
        keep.append(g)
      ga, gt = g.data_ptr(), codes[g.dtype]
    if c is not None:
      _check_tensor(c, f"copies[{i}]", (t.bfloat16,))
      if c.shape != p.shape or not c.is_contiguous():
        raise ValueError(f"copies[{i}] must be contiguous and have the shape "
                         f"{tuple(p.shape)} of its weight, got "
                         f"{tuple(c.shape)}")
      ca = c.data_ptr()
    rows.append((p.data_ptr(), ga, ca, p.numel(), codes[p.dtype], gt))
  table = table.copy()
  if rows:
    address, grad, copy, sizes, ptype, gtype = zip(*rows)
    if not np.array_equal(table["numel"], sizes):
      raise ValueError("the state was made for weights of other sizes")
    table["param"], table["grad"], table["copy"] = address, grad, copy
    table["param_type"], table["grad_type"] = ptype, gtype
    _check_apart(table)
  options = _native.AdamWOptions(
      beta_1=beta_1, beta_2=beta_2, epsilon=epsilon, weight_decay=weight_decay,
      grad_scale=1.0, step=1)
  rate, options.learning_rate_ptr = _device_scalar(learning_rate, t.float32)
  if rate is None:
    options.learning_rate = float(learning_rate)
  scale, options.grad_scale_ptr = _device_scalar(grad_scale, t.float32)
  if scale is None and grad_scale is not None:
    options.grad_scale = float(grad_scale)
  at, options.step_ptr = _device_scalar(step, t.int64)
  if at is None:
    options.step = state.step + 1 if step is None else int(step)
    if options.step < 1:
      raise ValueError(f"the first step is 1, got {options.step}")
  _native.adamw_update(table, state.as_struct(), options)
  del keep, rate, scale
  if at is None:
    state.step = int(options.step)
  return params


def _check_apart(table) -> None:
  """Two weights that share memory would be updated by two work-groups at
  once."""
  begin = table["param"].astype(np.int64)
  size = table["numel"] * np.where(
      table["param_type"] == _native.TYPE_F32, 4, 2)
  begin, size = begin[size > 0], size[size > 0]
  order = np.argsort(begin)
  begin, end = begin[order], (begin + size)[order]
  if (begin[1:] < end[:-1]).any():
    raise ValueError("two params share memory")


def adamw_moments(state: AdamWState):
  """(m, v) of a state as float32, laid out as state.m and state.v are; those
  of 32 bits are the state's own tensors."""
  if state.bits == 32:
    return state.m, state.v
  t = _native.require_gpu()
  m = t.empty(state.m.shape, dtype=t.float32, device=state.m.device)
  v = t.empty_like(m)
  _native.adamw_moments(state.as_struct(), m, v)
  return m, v
