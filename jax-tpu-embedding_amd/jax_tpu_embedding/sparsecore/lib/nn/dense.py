"""The dense operators of a ranking model that trains beside its tables.

No counterpart in the reference, whose users take these from their framework's
compiler. Families of hand-written gfx950 kernels behind the C ABI:

  layer_norm, layer_norm_grad
      layer norm of the activations that the lookups return, and its
      gradients, the weight's and the bias's included;
  sort_by_expert, tokens_to_experts, tokens_from_experts (and their _grad)
      a mixture of experts' tokens in the order of their experts and back,
      with the router's weights applied;
  expert_matmul, expert_matmul_grad
      the experts' layers between the two: products grouped by expert, whose
      numbers of rows stay on the GPU, and their gradients;
  quantize_weights, matmul_8bit
      the same products, or one plain product, in 8-bit floating point with a
      scale for each block of 128, for serving;
  gradient_norm, clip_gradients
      the global norm of all gradients, and gradients clipped to it;
  init_adamw_state, adamw_update, adamw_moments
      AdamW over all dense weights in one or a few launches, with moments in
      float32 or in 8 bits.

Arrays are torch tensors on the current GPU, work is enqueued on the current
stream and nothing waits for it; arguments that do not fit raise ValueError.
layer_norm, tokens_to_experts, expert_matmul and tokens_from_experts take part in
torch's autograd; the _grad functions are the same gradients for callers that keep
their own tape, as embedding.tpu_sparse_dense_matmul_grad's are. Nothing here
has forward-mode derivatives: tensors that carry a tangent are refused.
"""

from __future__ import annotations

from typing import NamedTuple

import numpy as np

from jax_tpu_embedding.sparsecore import _native

# Values that share a scale in 8-bit moments, and the most experts
# (SCEMB_ADAMW_BLOCK and SCEMB_MAX_EXPERTS).
ADAMW_BLOCK = 256
MAX_EXPERTS = 1024
# Values that share a scale in 8-bit products, along each dimension
# (SCEMB_BLOCK_8BIT).
BLOCK_8BIT = 128

_binding = None


def _calls():
  """The native module of the calls, once a GPU has been seen."""
  global _binding
  if _binding is None:
    _native.require_gpu()
    _binding = _native.dense_binding()
  return _binding


_workspace = _native.WORKSPACE.get

_functions = {}


def _function(name: str):
  """The autograd functions, made on first use: torch is imported late."""
  if not _functions:
    t = _native.torch()
    once = t.autograd.function.once_differentiable

    class LayerNorm(t.autograd.Function):

      @staticmethod
      def forward(ctx, x, weight, bias, epsilon):
        y, mean, rstd = _calls().layer_norm(x, weight, bias, epsilon, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_f32 = bias is not None and bias.dtype == t.float32
        ctx.mark_non_differentiable(mean, rstd)
        return y, mean, rstd

      @staticmethod
      @once
      def backward(ctx, y_grad, *_):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _calls().layer_norm_grad(
            y_grad, x, mean, rstd, weight, need[1], need[2], ctx.bias_f32,
            _workspace)
        return dx if need[0] else None, dw, db, None

    class ToExperts(t.autograd.Function):

      @staticmethod
      def forward(ctx, x, positions, offsets):
        ctx.save_for_backward(positions, offsets)
        return _calls().tokens_to_experts(x, positions, offsets)

      @staticmethod
      @once
      def backward(ctx, rows_grad):
        dx = _calls().tokens_from_experts(rows_grad, None, *ctx.saved_tensors,
                                          "rows_grad")
        return dx, None, None

    class FromExperts(t.autograd.Function):

      @staticmethod
      def forward(ctx, rows, weights, positions, offsets):
        ctx.save_for_backward(rows, weights, positions, offsets)
        return _calls().tokens_from_experts(rows, weights, positions, offsets,
                                            "rows")

      @staticmethod
      @once
      def backward(ctx, y_grad):
        need = ctx.needs_input_grad
        drows, dw = _calls().tokens_from_experts_grad(y_grad,
                                                      *ctx.saved_tensors)
        return (drows if need[0] else None, dw if need[1] else None, None,
                None)

    class Product(t.autograd.Function):

      @staticmethod
      def forward(ctx, rows, weights, offsets):
        ctx.save_for_backward(rows, weights, offsets)
        return _calls().expert_matmul(rows, weights, offsets, _workspace)

      @staticmethod
      @once
      def backward(ctx, y_grad):
        rows, weights, offsets = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*_calls().expert_matmul_grad(y_grad, rows, weights, offsets,
                                             need[0], need[1], _workspace),
                None)

    _functions.update(norm=LayerNorm, to=ToExperts, back=FromExperts,
                      product=Product)
  return _functions[name]


# ---------------------------------------------------------------------------
# Layer norm.
# ---------------------------------------------------------------------------


def layer_norm(x, weight=None, bias=None, *, epsilon: float = 1e-6,
               return_stats: bool = False):
  """Layer norm of x over its last dimension, of x's type.

  x: float32, bfloat16 or float16, [..., dim]; any strides (rows that are not
    contiguous in the last dimension are copied first).
  weight, bias: [dim], float32 or x's type, the same for both; None: one, zero.
  epsilon: added to the variance.
  return_stats: also return the float32 mean and reciprocal deviation of every
    row ([...]), which layer_norm_grad takes. They are constants to autograd:
    no gradient flows through them.

  Statistics and products are float32; the result is rounded once. The mean's
  own rounding is taken out of the result, so a row of one value gives the bias
  whatever that value is. A row that holds an infinity or a NaN gives a row of
  NaN.
  """
  calls = _calls()
  if calls.wants_grad(x, weight, bias):
    out = _function("norm").apply(x, weight, bias, epsilon)
    return out if return_stats else out[0]
  return calls.layer_norm(x, weight, bias, epsilon, bool(return_stats))


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
  return _calls().layer_norm_grad(y_grad, x, mean, rstd, weight, True,
                                  bool(with_bias), True, _workspace)


# ---------------------------------------------------------------------------
# Tokens and experts.
# ---------------------------------------------------------------------------


class ExpertOrder(NamedTuple):
  """The order of tokens' choices by expert, int32 tensors on the GPU, as
  sort_by_expert makes it. To drop a choice, sort with an id out of range:
  positions that are changed afterwards leave a row without a choice, and what
  is written row by row (tokens_to_experts, the gradient of
  tokens_from_experts's rows) is undefined there.

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
  return ExpertOrder(*_calls().sort_by_expert(expert_ids, num_experts,
                                              _workspace))


def tokens_to_experts(x, order: ExpertOrder):
  """The tokens' rows in the order of their experts, [choices in all, dim]:
  row order.positions[t, k] is x[t]; rows of dropped choices are zero.

  x: [tokens, dim], float32, bfloat16 or float16.
  """
  calls = _calls()
  if calls.wants_grad(x):
    return _function("to").apply(x, order.positions, order.offsets)
  return calls.tokens_to_experts(x, order.positions, order.offsets)


def tokens_to_experts_grad(rows_grad, order: ExpertOrder):
  """The gradient of tokens_to_experts's x: the sum of the gradients of its
  choices' rows, in float32, rounded once. Rows of dropped choices are not
  read."""
  return _calls().tokens_from_experts(rows_grad, None, order.positions,
                                      order.offsets, "rows_grad")


def tokens_from_experts(rows, weights, order: ExpertOrder):
  """The experts' rows back at their tokens, [tokens, dim]: the sum over the
  token's choices of weight * row, in float32, rounded once.

  rows: [choices in all, dim]; rows of dropped choices are not read and add
    nothing (a token without choices gets zeros).
  weights: of the ids' shape, float32 or rows' type; None: one.
  """
  calls = _calls()
  if calls.wants_grad(rows, weights):
    return _function("back").apply(rows, weights, order.positions,
                                   order.offsets)
  return calls.tokens_from_experts(rows, weights, order.positions,
                                   order.offsets, "rows")


def tokens_from_experts_grad(y_grad, rows, weights, order: ExpertOrder):
  """Gradients of tokens_from_experts: (of rows, of weights).

  Rows of dropped choices get zeros, and so do their weights. The second is
  None without weights.
  """
  return _calls().tokens_from_experts_grad(y_grad, rows, weights,
                                           order.positions, order.offsets)


def expert_matmul(rows, weights, order: ExpertOrder):
  """Every expert's rows times its weights, [choices in all, outer]: row r of
  expert e is rows[r] @ weights[e].

  rows: [choices in all, inner] in the order of their experts, as
    tokens_to_experts returns them; float32, bfloat16 or float16. Rows of
    dropped choices are not read and give zeros.
  weights: [experts, inner, outer] of rows' type. Either of the last two
    dimensions may be the contiguous one (others are copied first), so weights
    stored by output are given as their transpose.
  order: sort_by_expert's; only its offsets are used, on the GPU: nothing waits
    for the experts' numbers of rows. With a part of the offsets, and of the
    weights, it is the product of some experts: rows of the others are not read
    and give zeros.

  Sums are float32, rounded once. float32 products are exact to float32's own
  rounding (no shortened operands). Calls of more than about 2^24 tiles (of 32 x
  128 values of the result, or larger ones) are refused.
  """
  calls = _calls()
  if calls.wants_grad(rows, weights):
    return _function("product").apply(rows, weights, order.offsets)
  return calls.expert_matmul(rows, weights, order.offsets, _workspace)


def expert_matmul_grad(y_grad, rows, weights, order: ExpertOrder, *,
                       with_rows: bool = True, with_weights: bool = True):
  """Gradients of expert_matmul: (of rows, of weights), of their types; None
  for one that is not wanted.

  Rows of dropped choices get zeros, and so do the weights of an expert without
  rows. The weights' gradient is laid out in memory as the weights are; its sum
  over the rows is float32, in an order that the sizes and the order decide.
  """
  return _calls().expert_matmul_grad(y_grad, rows, weights, order.offsets,
                                     bool(with_rows), bool(with_weights),
                                     _workspace)


class Weights8(NamedTuple):
  """Weights in 8 bits, as quantize_weights makes them: what a server keeps.

  codes: float8_e4m3fn, [(experts,) outer, inner rounded up to BLOCK_8BIT]: the
    inner dimension one after another, zeros behind it.
  exponents: int32, [(experts,) blocks of outer, blocks of inner]: a value is
    its code times 2^(exponent - 127).
  inner: the inner dimension.
  """

  codes: object
  exponents: object
  inner: int


def quantize_weights(weights) -> Weights8:
  """Weights for matmul_8bit, once.

  weights: [inner, outer] or [experts, inner, outer], float32, bfloat16 or
    float16, any strides; inner at most 2^22.

  BLOCK_8BIT x BLOCK_8BIT values share a scale, the least power of two (2^-126
  at least) with no magnitude of the block above 448 times it; values are
  rounded to the nearest code, which is 2^-4 of the value off at most (2^-10 of
  the scale where that is more). A block that holds an infinity or a NaN is NaN
  throughout. Autograd does not follow the codes.
  """
  inner = weights.shape[-2] if getattr(weights, "ndim", 0) >= 2 else 0
  return Weights8(*_calls().quantize_weights(weights), inner)


def matmul_8bit(rows, weights: Weights8, order: ExpertOrder | None = None):
  """rows @ weights in 8-bit floating point, of rows' type, for serving: there
  are no gradients, and rows that autograd would follow are refused.

  rows: [rows, inner], float32, bfloat16 or float16. They are brought to 8 bits
    in the call, as the weights are, but with a scale for each BLOCK_8BIT
    neighbours of a row.
  weights: quantize_weights's; of several experts with an order, else of none.
  order: sort_by_expert's, for rows in the order of their experts as
    tokens_to_experts returns them; rows of dropped choices are not read and
    give zeros.

  Products of codes are exact, summed in float32 and rounded once. A row that
  holds an infinity or a NaN gives a row of NaN. The limit on tiles is
  expert_matmul's.
  """
  calls = _calls()
  if calls.wants_grad(rows):
    raise ValueError("matmul_8bit has no gradients: call it under "
                     "torch.no_grad(), or detach the rows")
  return calls.matmul_8bit(rows, weights.codes, weights.exponents,
                           weights.inner,
                           None if order is None else order.offsets,
                           _workspace)


# ---------------------------------------------------------------------------
# AdamW.
# ---------------------------------------------------------------------------

# scemb_adamw_tensor_t; a state keeps each weight's size and decay in it, the
# native module fills in the rest.
_TENSOR = np.dtype([
    ("param", np.uint64), ("grad", np.uint64), ("copy", np.uint64),
    ("numel", np.int64), ("param_type", np.int32), ("grad_type", np.int32),
    ("decay", np.int32), ("reserved", np.int32)])


class AdamWState:
  """The moments of a list of weights, and the steps taken.

  m, v: the moments of all weights in one tensor each, weight i's from
    first[i] on, first[i] being a multiple of ADAMW_BLOCK. float32, or int8 and
    uint8 with 8 bits, whose values adamw_moments returns.
  m_scale, v_scale: with 8 bits, a float32 for each ADAMW_BLOCK values; else
    None.
  step: updates made so far, where the host counts them. Updates whose step is a
    value on the GPU are not in it: that value is the count.
  bits: 8 or 32.

  A checkpoint keeps these tensors and the step (the value on the GPU, where
  that counts); a state made for the same weights takes them back with copy_()
  and `state.step = ...`.
  """

  def __init__(self, sizes, decay, bits: int):
    t = _native.torch()
    padded = -(-np.asarray(sizes, np.int64) // ADAMW_BLOCK) * ADAMW_BLOCK
    ends = np.cumsum(padded)
    total = int(ends[-1]) if len(sizes) else 0
    self.first = (ends - padded).tolist()
    self.bits = bits
    self.step = 0
    new = lambda n, dtype: t.zeros(n, dtype=dtype, device=_native.device())
    if bits == 8:
      self.m, self.v = new(total, t.int8), new(total, t.uint8)
      self.m_scale = new(total // ADAMW_BLOCK, t.float32)
      self.v_scale = new(total // ADAMW_BLOCK, t.float32)
    else:
      self.m, self.v = new(total, t.float32), new(total, t.float32)
      self.m_scale = self.v_scale = None
    # What steps with hyperparameters on the GPU make of them.
    self._scratch = new(4, t.float32)
    layout = np.zeros(len(sizes), _TENSOR)
    layout["numel"] = sizes
    layout["decay"] = decay
    self._layout = layout.tobytes()

  @property
  def step(self) -> int:
    return self._step

  @step.setter
  def step(self, value: int):
    self._step = value
    # Whether the last update's step was a value on the GPU: the host cannot
    # count on from `step` then.
    self._counted_on_gpu = False


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
  sizes = _calls().adamw_sizes(params)
  decay = [True] * len(sizes) if decay is None else [bool(d) for d in decay]
  if len(decay) != len(sizes):
    raise ValueError(f"decay has {len(decay)} entries for {len(sizes)} "
                     "params")
  return AdamWState(sizes, decay, state_bits)


def _scalar(x, is_int, missing):
  """(host value, None, None) of a number, (missing, its address, a tensor to
  keep until the launch) of a single value on the GPU."""
  if x is None:
    return missing, None, None
  t = _native.torch()
  if not isinstance(x, t.Tensor) or not x.is_cuda:
    return x, None, None
  x = _calls().adamw_scalar(x, is_int)
  return missing, x.data_ptr(), x


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
    the rounded weight: the working copies of float32 weights. Params and
    copies may not share memory, but a bfloat16 weight may be its own copy.
    Gradients may not share memory with another weight or a copy; that is not
    checked.
  step: None (state.step + 1), an int, or a single int64 on the GPU, which a
    captured graph advances itself (what the host gives, this and every other
    hyperparameter, is the same in all replays). The first step is 1. After an
    update with a value on the GPU, None is refused until an int is given here
    or set as state.step.
  """
  if not (0 <= beta_1 < 1 and 0 <= beta_2 < 1 and epsilon >= 0):
    raise ValueError("beta_1 and beta_2 must be within [0, 1) and epsilon not "
                     f"negative, got {beta_1}, {beta_2} and {epsilon}")
  # pylint: disable=protected-access
  if step is None and state._counted_on_gpu:
    raise ValueError("the state's updates were counted on the GPU: give the "
                     "step, or set state.step to the updates made so far")
  rate, rate_at, keep_rate = _scalar(learning_rate, False, 0.0)
  scale, scale_at, keep_scale = _scalar(grad_scale, False, 1.0)
  at, step_at, keep_step = _scalar(step, True, state.step + 1)
  at = int(at)
  if step_at is None and at < 1:
    raise ValueError(f"the first step is 1, got {at}")
  _calls().adamw_update(
      params, grads, copies, state._layout, state.m, state.v,
      state.m_scale, state.v_scale, state._scratch, float(rate), beta_1,
      beta_2, epsilon, weight_decay, float(scale), at, rate_at, step_at,
      scale_at)
  del keep_rate, keep_scale, keep_step
  if step_at is None:
    state.step = at
  else:
    state._counted_on_gpu = True
  return params


def adamw_moments(state: AdamWState):
  """(m, v) of a state as float32, laid out as state.m and state.v are; those
  of 32 bits are the state's own tensors."""
  if state.bits == 32:
    return state.m, state.v
  return _calls().adamw_moments(state.m, state.v, state.m_scale,
                                state.v_scale)


# ---------------------------------------------------------------------------
# The gradients' norm.
# ---------------------------------------------------------------------------


def gradient_norm(grads, *, max_norm: float | None = None):
  """The norm of all values of all gradients, sqrt(sum of g^2), a single
  float32 on the GPU; with max_norm (norm, factor), the factor being
  min(1, max_norm / norm), which adamw_update takes as grad_scale: gradients
  clipped to a global norm without a pass that writes them.

  grads: a sequence of float32, bfloat16 or float16 tensors of any shapes and
    strides, or None (left out). What is given twice counts twice. No gradients
    flow through the norm: tensors that autograd would follow (made with
    create_graph) are refused, unless under torch.no_grad().
  max_norm: not negative.

  Squares are summed in 64 bits, in an order that the sizes decide. With an
  infinity among the values the norm is infinite and the factor 0, with a NaN
  both are NaN.
  """
  norm, factor = _calls().gradient_norm(grads, max_norm, _workspace)
  return norm if max_norm is None else (norm, factor)


def clip_gradients(grads, max_norm: float):
  """Scales all gradients, in place, by min(1, max_norm / their norm); returns
  the norm that they had, a single float32 on the GPU.

  grads: as for gradient_norm, but tensors have to be without gaps in memory
    (any order of dimensions) and share none.

  Products are float32, rounded once. Gradients whose norm is within max_norm
  are not written. With an infinity among the values the factor is 0 (and the
  infinities become NaN), with a NaN all values become NaN.
  """
  return _calls().clip_gradients(grads, max_norm, _workspace)
