"""The dense operators that train and serve beside the tables, as timed cases.

A ranking model does three things with what the lookups return: it normalises
the concatenated activations, it sends every sample to a few of many experts
and adds their answers, and it updates the dense weights. Each case is one
pass through the public entry points of
`jax_tpu_embedding.sparsecore.lib.nn.dense`:

  norm            dense.layer_norm of a matrix of activations
  norm_grad       dense.layer_norm_grad: the gradients of the activations, of
                  the weight and of the bias
  to_experts      dense.sort_by_expert of the chosen experts, then
                  dense.tokens_to_experts: the tokens' rows, expert by expert
  to_experts_grad      dense.tokens_to_experts_grad
  from_experts         dense.tokens_from_experts: the experts' rows back at
                       their tokens, weighted and added
  from_experts_grad    dense.tokens_from_experts_grad: the gradients of the
                       experts' rows and of the weights
  adamw           dense.adamw_update of all dense weights, with moments in 32
                  bits or in 8

With `own` false the same is computed by elementary tensor operations in 32
bits, rounded once to the outputs' types.
"""

import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for _p in (ROOT, os.path.join(ROOT, "jax-tpu-embedding_amd")):
  if _p not in sys.path:
    sys.path.insert(0, _p)

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

EPSILON = 1e-6  # layer norm
BLOCK = 256  # values that share a scale in 8-bit moments
RATE, BETA_1, BETA_2, ADAM_EPSILON, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01


def listed():
  return [
      # One online request: the activations of a few candidates, one feature
      # of 128 columns. Latency.
      dict(name="norm_request", kind="norm", rows=64, dim=128, dtype="f32",
           weight="f32", stats=False),
      # The benchmark's 26 features of 128 columns side by side.
      dict(name="norm_large", kind="norm", rows=65536, dim=3328,
           dtype="bf16", weight="f32", stats=True),
      # The same batch after a projection to 1024 columns, backwards.
      dict(name="norm_grad_large", kind="norm_grad", rows=65536, dim=1024,
           dtype="bf16", weight="f32"),
      # An odd batch of one narrow feature (100 columns).
      dict(name="norm_grad_odd", kind="norm_grad", rows=20011, dim=100,
           dtype="f32", weight="f32"),
      # One online request through a small mixture of experts. Latency.
      dict(name="to_experts_request", kind="to_experts", tokens=64,
           experts=8, choices=2, dim=128, dtype="f32", dropped=0.0),
      # A whole training batch, 64 experts, two for each token.
      dict(name="to_experts_large", kind="to_experts", tokens=65536,
           experts=64, choices=2, dim=1024, dtype="bf16", dropped=0.0),
      dict(name="from_experts_large", kind="from_experts", tokens=65536,
           experts=64, choices=2, dim=1024, dtype="bf16", dropped=0.0),
      # A smaller batch, more choices, some of them dropped.
      dict(name="from_experts_grad", kind="from_experts_grad", tokens=16384,
           experts=32, choices=4, dim=512, dtype="bf16", dropped=0.05),
      dict(name="to_experts_grad_odd", kind="to_experts_grad", tokens=20011,
           experts=61, choices=3, dim=100, dtype="f32", dropped=0.05),
      # A small tower that trains in bfloat16.
      dict(name="adamw_small", kind="adamw", tensors=12, smallest=1,
           largest=16384, dtype="bf16", grad="bf16", copies=False, bits=8),
      # A large tower in float32.
      dict(name="adamw_32", kind="adamw", tensors=60, smallest=128,
           largest=33_554_432, dtype="f32", grad="f32", copies=False,
           bits=32),
      # The same with bfloat16 gradients and working copies, small moments.
      dict(name="adamw_8", kind="adamw", tensors=24, smallest=100,
           largest=33_554_432, dtype="f32", grad="bf16", copies=True, bits=8),
  ]


def _log_int(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
  """One more case of the same ranges, no dearer than the largest above."""
  while True:
    kind = rng.choice(["norm", "norm_grad", "to_experts", "to_experts_grad",
                       "from_experts", "from_experts_grad", "adamw", "adamw"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind in ("norm", "norm_grad"):
      dim = rng.choice([_log_int(rng, 8, 16384), _log_int(rng, 8, 16384),
                        64, 128, 256, 512, 1024, 2048, 4096])
      c = dict(kind=kind, rows=_log_int(rng, 16, 262144), dim=dim,
               dtype=dtype, weight=rng.choice(["f32", dtype]))
      if kind == "norm":
        c["stats"] = rng.random() < 0.5
      if c["rows"] * dim <= 200_000_000:
        return c
    elif kind == "adamw":
      dtype = rng.choice(["f32", "f32", "bf16"])
      c = dict(kind=kind, tensors=_log_int(rng, 2, 300),
               smallest=_log_int(rng, 1, 4096),
               largest=_log_int(rng, 4096, 33_554_432), dtype=dtype,
               grad=rng.choice([dtype, "bf16"]),
               copies=dtype == "f32" and rng.random() < 0.4,
               bits=rng.choice([8, 32]))
      if sum(_sizes(c)) <= 150_000_000:
        return c
    else:
      experts = _log_int(rng, 2, 256)
      c = dict(kind=kind, tokens=_log_int(rng, 16, 131072), experts=experts,
               choices=min(experts, rng.choice([1, 2, 2, 4, 6, 8])),
               dim=rng.choice([_log_int(rng, 8, 4096), 64, 128, 256, 512,
                               1024, 2048]),
               dtype=dtype, dropped=rng.choice([0.0, 0.05, 0.3]))
      if c["tokens"] * c["choices"] * c["dim"] <= 130_000_000:
        return c


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------


def _sizes(case):
  """Values of each weight, from the smallest to the largest, odd ones."""
  n, lo, hi = case["tensors"], case["smallest"], case["largest"]
  step = math.log(hi / lo) / (n - 1)
  sizes = [int(round(lo * math.exp(step * i))) for i in range(n)]
  return [max(1, v - 1) if i % 4 == 1 else v for i, v in enumerate(sizes)]


def _generator(seed):
  g = torch.Generator(device="cuda")
  g.manual_seed(seed * 2 + 1)
  return g


def _randn(shape, g, dtype=torch.float32, scale=1.0):
  x = torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g)
  return x.to(dtype)


def _prepare_norm(case, g):
  rows, dim = case["rows"], case["dim"]
  dtype, wtype = DTYPES[case["dtype"]], DTYPES[case["weight"]]
  # Activations with a scale and a mean of each row's own.
  x = torch.empty((rows, dim), device="cuda").normal_(generator=g)
  x.mul_(_randn((rows, 1), g).mul_(0.5).exp_()).add_(_randn((rows, 1), g))
  s = {"x": x.to(dtype),
       "weight": (1.0 + _randn((dim,), g, scale=0.1)).to(wtype),
       "bias": _randn((dim,), g, wtype, 0.1)}
  if case["kind"] == "norm":
    s["stats"] = case["stats"]
  else:
    del x
    s["y_grad"] = _randn((rows, dim), g, dtype)
    _, s["mean"], s["rstd"] = _norm(s["x"], s["weight"], s["bias"])
  return s


def _prepare_experts(case, g):
  t, e, k, d = (case[n] for n in ("tokens", "experts", "choices", "dim"))
  dtype = DTYPES[case["dtype"]]
  # A router's scores: some experts are liked more than others.
  scores = _randn((t, e), g) + _randn((1, e), g)
  top, ids = scores.topk(k, dim=1)
  # Choices that an expert's capacity or a padded sample drops.
  ids[torch.rand((t, k), device="cuda", generator=g) < case["dropped"]] = -1
  s = {"ids": ids, "experts": e}
  if case["kind"] == "to_experts":
    s["x"] = _randn((t, d), g, dtype)
    return s
  s["positions"], s["sources"], s["offsets"] = _sort(ids, e)
  if case["kind"] != "from_experts_grad":
    s["rows"] = _randn((t * k, d), g, dtype)
  if case["kind"] != "to_experts_grad":
    s["weights"] = top.softmax(1)
  if case["kind"] == "from_experts_grad":
    s["rows"] = _randn((t * k, d), g, dtype)
    s["y_grad"] = _randn((t, d), g, dtype)
  return s


def _prepare_adamw(case, g):
  """Weights and gradients in one buffer each, as gradient buckets are; every
  weight starts at a multiple of BLOCK, and so do its moments. The moments
  are those of a run under way."""
  sizes, dtype = _sizes(case), DTYPES[case["dtype"]]
  first, total = [], 0
  for n in sizes:
    first.append(total)
    total += -(-n // BLOCK) * BLOCK
  used = torch.zeros(total, dtype=torch.bool, device="cuda")
  decays = torch.zeros((total // BLOCK, 1), device="cuda")
  for i, (at, n) in enumerate(zip(first, sizes)):
    used[at:at + n] = True
    decays[at // BLOCK:-(-(at + n) // BLOCK)] = i % 3 > 0
  # Gradients differ in size from block to block.
  scale = _randn((total // BLOCK, 1), g).exp_().mul_(1e-3).expand(-1, BLOCK)
  scale = scale.reshape(-1) * used
  s = {"p": (_randn(total, g, scale=0.02) * used).to(dtype),
       "g": (_randn(total, g) * scale).to(DTYPES[case["grad"]]),
       "copies": (torch.zeros(total, dtype=torch.bfloat16, device="cuda")
                  if case["copies"] else None),
       "bits": case["bits"], "decays": decays, "step": 1000,
       "grad_scale": torch.full((), 0.5, device="cuda")}
  m = _randn(total, g) * scale * 0.3
  v = (_randn(total, g) * scale).square_() + scale.square() * 0.1
  cut = lambda x: [x[at:at + n] for at, n in zip(first, sizes)]
  s["params"], s["grads"] = cut(s["p"]), cut(s["g"])
  if case["bits"] == 8:
    s["m"], s["m_scale"] = _encode_m(m.view(-1, BLOCK))
    s["v"], s["v_scale"] = _encode_r(v.sqrt_().view(-1, BLOCK))
  else:
    s["m"], s["v"] = m, v
  if own:
    from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top

    state = dense.init_adamw_state(
        s["params"], state_bits=case["bits"],
        decay=[i % 3 > 0 for i in range(len(sizes))])
    for name in ("m", "v", "m_scale", "v_scale"):
      if name in s:
        getattr(state, name).copy_(s[name].view(-1))
    state.step = s["step"]
    s["state"] = state
    s["working"] = cut(s["copies"]) if case["copies"] else None
  return s


def prepare(case, seed):
  g = _generator(seed)
  if case["kind"].startswith("norm"):
    s = _prepare_norm(case, g)
  elif case["kind"] == "adamw":
    s = _prepare_adamw(case, g)
  else:
    s = _prepare_experts(case, g)
  s["kind"] = case["kind"]
  return s


# ---------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------


def _norm(x, weight, bias):
  xf = x.float()
  mean = xf.mean(1, keepdim=True)
  xf = xf - mean
  rstd = torch.rsqrt((xf * xf).mean(1, keepdim=True) + EPSILON)
  y = xf * rstd * weight.float() + bias.float()
  return y.to(x.dtype), mean.view(-1), rstd.view(-1)


def _norm_grad(y_grad, x, mean, rstd, weight):
  rstd = rstd.unsqueeze(1)
  dy = y_grad.float()
  xhat = (x.float() - mean.unsqueeze(1)) * rstd
  wdy = dy * weight.float()
  along = (wdy * xhat).mean(1, keepdim=True)
  dx = (wdy - wdy.mean(1, keepdim=True) - xhat * along) * rstd
  dw = (dy * xhat).sum(0)
  db = dy.sum(0)
  return dx.to(x.dtype), dw.to(weight.dtype), db.to(weight.dtype)


def _sort(ids, experts):
  """Positions of the choices in the order of their experts (dropped ones at
  the end), the choice at each position, and where each expert begins."""
  flat = ids.reshape(-1)
  key = torch.where((flat >= 0) & (flat < experts), flat, experts)
  key, sources = torch.sort(key, stable=True)
  positions = torch.empty_like(sources)
  positions[sources] = torch.arange(flat.numel(), device=flat.device)
  offsets = torch.searchsorted(
      key, torch.arange(experts + 1, device=flat.device))
  return (positions.to(torch.int32).view(ids.shape), sources.to(torch.int32),
          offsets.to(torch.int32))


def _to_experts(x, sources, offsets, choices):
  kept = torch.arange(sources.numel(), device=x.device) < offsets[-1]
  return torch.where(kept.unsqueeze(1), x[(sources // choices).long()], 0)


def _of_tokens(rows, positions, offsets):
  """[tokens, choices, dim]: the rows of each token's choices, zero for those
  that were dropped."""
  kept = positions < offsets[-1]
  return torch.where(kept.unsqueeze(2), rows[positions.long()].float(), 0.0)


def _to_experts_grad(rows, positions, offsets):
  return _of_tokens(rows, positions, offsets).sum(1).to(rows.dtype)


def _from_experts(rows, weights, positions, offsets):
  picked = _of_tokens(rows, positions, offsets)
  return (picked * weights.unsqueeze(2)).sum(1).to(rows.dtype)


def _from_experts_grad(y_grad, rows, weights, positions, offsets):
  dy = y_grad.float().unsqueeze(1)
  dw = (_of_tokens(rows, positions, offsets) * dy).sum(2)
  kept = (positions < offsets[-1]).unsqueeze(2)
  drows = torch.empty_like(rows)
  drows[positions.reshape(-1).long()] = torch.where(
      kept, weights.unsqueeze(2) * dy, 0.0).to(rows.dtype).view(
          -1, rows.shape[1])
  return drows, dw


def _encode_m(m):
  """Blocks of first moments as (8 bits each, scale): the value of q is
  scale * (q / 127) * |q / 127|."""
  scale = m.abs().amax(1, keepdim=True)
  q = (m.abs() / torch.where(scale > 0, scale, 1.0)).sqrt() * 127.0
  return torch.where(m < 0, -q.round(), q.round()).to(torch.int8), scale


def _encode_r(r):
  """The same for roots of second moments, which are positive: the root of q
  is scale * (q / 255)^2, and only an exact zero has q = 0."""
  scale = r.amax(1, keepdim=True)
  q = ((r / torch.where(scale > 0, scale, 1.0)).sqrt() * 255.0).round()
  return torch.maximum(q, (r > 0).float()).to(torch.uint8), scale


def _decode_m(q, scale):
  q = q.float() * (1.0 / 127.0)
  return q * q.abs() * scale


def _decode_v(q, scale):
  q = q.float() * (1.0 / 255.0)
  r = q * q * scale
  return r * r


def _adamw(s):
  s["step"] += 1
  p = s["p"].float().view(-1, BLOCK)
  g = s["g"].float().view(-1, BLOCK) * s["grad_scale"]
  if s["bits"] == 8:
    m = _decode_m(s["m"], s["m_scale"])
    v = _decode_v(s["v"], s["v_scale"])
  else:
    m, v = s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK)
  m = m * BETA_1 + g * (1.0 - BETA_1)
  v = v * BETA_2 + g * g * (1.0 - BETA_2)
  r = v.sqrt()
  rate = RATE / (1.0 - BETA_1 ** s["step"])
  root = 1.0 / math.sqrt(1.0 - BETA_2 ** s["step"])
  p = p * (1.0 - s["decays"] * (RATE * DECAY)) - m / (
      r * root + ADAM_EPSILON) * rate
  s["p"].view(-1, BLOCK).copy_(p)
  out = {"p": s["p"]}
  if s["copies"] is not None:
    s["copies"].view(-1, BLOCK).copy_(p)
    out["copies"] = s["copies"]
  if s["bits"] == 8:
    s["m"], s["m_scale"] = _encode_m(m)
    s["v"], s["v_scale"] = _encode_r(r)
    out["m"] = _decode_m(s["m"], s["m_scale"]).view(-1)
    out["v"] = _decode_v(s["v"], s["v_scale"]).view(-1)
  else:
    s["m"].view(-1, BLOCK).copy_(m)
    s["v"].view(-1, BLOCK).copy_(v)
    out["m"], out["v"] = s["m"], s["v"]
  return out


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------


def _run_plain(s):
  kind = s["kind"]
  if kind == "norm":
    got = _norm(s["x"], s["weight"], s["bias"])
    return got if s["stats"] else got[:1]
  if kind == "norm_grad":
    return _norm_grad(s["y_grad"], s["x"], s["mean"], s["rstd"], s["weight"])
  if kind == "to_experts":
    positions, sources, offsets = _sort(s["ids"], s["experts"])
    rows = _to_experts(s["x"], sources, offsets, s["ids"].shape[1])
    return rows, positions, sources, offsets
  if kind == "to_experts_grad":
    return _to_experts_grad(s["rows"], s["positions"], s["offsets"])
  if kind == "from_experts":
    return _from_experts(s["rows"], s["weights"], s["positions"],
                         s["offsets"])
  if kind == "from_experts_grad":
    return _from_experts_grad(s["y_grad"], s["rows"], s["weights"],
                              s["positions"], s["offsets"])
  return _adamw(s)


def _run_own(s):
  from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top

  kind = s["kind"]
  if kind == "norm":
    if s["stats"]:
      return dense.layer_norm(s["x"], s["weight"], s["bias"],
                              epsilon=EPSILON, return_stats=True)
    return (dense.layer_norm(s["x"], s["weight"], s["bias"],
                             epsilon=EPSILON),)
  if kind == "norm_grad":
    return dense.layer_norm_grad(s["y_grad"], s["x"], s["mean"], s["rstd"],
                                 s["weight"])
  if kind == "to_experts":
    order = dense.sort_by_expert(s["ids"], s["experts"])
    rows = dense.tokens_to_experts(s["x"], order)
    return rows, order.positions, order.sources, order.offsets
  if kind == "adamw":
    dense.adamw_update(
        s["params"], s["grads"], s["state"], learning_rate=RATE,
        beta_1=BETA_1, beta_2=BETA_2, epsilon=ADAM_EPSILON,
        weight_decay=DECAY, grad_scale=s["grad_scale"], copies=s["working"])
    out = {"p": s["p"]}
    if s["copies"] is not None:
      out["copies"] = s["copies"]
    out["m"], out["v"] = dense.adamw_moments(s["state"])
    return out
  order = dense.ExpertOrder(positions=s["positions"], sources=s["sources"],
                            offsets=s["offsets"])
  if kind == "to_experts_grad":
    return dense.tokens_to_experts_grad(s["rows"], order)
  if kind == "from_experts":
    return dense.tokens_from_experts(s["rows"], s["weights"], order)
  return dense.tokens_from_experts_grad(s["y_grad"], s["rows"], s["weights"],
                                        order)


def run(state):
  return _run_own(state) if own else _run_plain(state)


def work(case):
  kind = case["kind"]
  size = lambda name: 4 if case[name] == "f32" else 2
  if kind.startswith("norm"):
    n, d = case["rows"] * case["dim"], case["dim"]
    if kind == "norm":
      stats = 8 * case["rows"] if case["stats"] else 0
      return {"bytes": 2 * n * size("dtype") + 2 * d * size("weight") + stats,
              "flops": 8 * n}
    return {"bytes": 3 * n * size("dtype") + 3 * d * size("weight") +
            8 * case["rows"], "flops": 14 * n}
  if kind == "adamw":
    n = sum(_sizes(case))
    each = 2 * size("dtype") + size("grad") + 2 * case["copies"]
    # Moments read and written; those in 8 bits are returned as values too.
    each += 16 if case["bits"] == 32 else 4 + 8 + 2 * 2 * 4 / BLOCK
    return {"bytes": n * each, "flops": 20 * n}
  t, k, d = case["tokens"], case["choices"], case["dim"]
  n, b = t * k, size("dtype")
  if kind == "to_experts":
    return {"bytes": (t + n) * d * b + n * (8 + 4 + 4) +
            4 * (case["experts"] + 1), "flops": 4 * n}
  if kind == "to_experts_grad":
    return {"bytes": (t + n) * d * b + 4 * n, "flops": n * d}
  if kind == "from_experts":
    return {"bytes": (t + n) * d * b + 8 * n, "flops": 2 * n * d}
  return {"bytes": (t + 2 * n) * d * b + 12 * n, "flops": 3 * n * d}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.
# ---------------------------------------------------------------------------


def _exact_norm(s, grad):
  x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
  if not grad:
    var, mean = torch.var_mean(x, 1, correction=0)
    rstd = (var + EPSILON).pow(-0.5)
    y = torch.addcmul(b, (x - mean[:, None]).mul_(rstd[:, None]), w)
    return (y, mean, rstd) if s["stats"] else (y,)
  # As a function of the statistics that were handed over: the gradient is
  # what is left of w * dy without its parts along 1 and along xhat.
  d = x.shape[1]
  xhat = torch.addcmul(-(s["mean"].double() * s["rstd"].double())[:, None],
                       x, s["rstd"].double()[:, None])
  dy = s["y_grad"].double()
  dw = torch.einsum("rc,rc->c", dy, xhat)
  db = torch.ones(1, x.shape[0], dtype=x.dtype, device=x.device).mm(dy)[0]
  h = dy * w
  a = h.sum(1) / d
  c = torch.einsum("rc,rc->r", h, xhat) / d
  dx = torch.addcmul(h - a[:, None], xhat, c[:, None], value=-1.0)
  return dx.mul_(s["rstd"].double()[:, None]), dw, db


def _exact_experts(s):
  kind = s["kind"]
  if kind == "to_experts":
    x, ids = s["x"], s["ids"].cpu()
    t, k = ids.shape
    # Where each choice goes: choices before it of lower or equal expert.
    key = ids.reshape(-1).clone()
    key[(key < 0) | (key >= s["experts"])] = s["experts"]
    where = torch.from_numpy(key.numpy().argsort(kind="stable")).cuda()
    rows = x.double().repeat_interleave(k, 0)
    rows[key.cuda() == s["experts"]] = 0.0
    return rows.index_select(0, where), None, None, None
  pos = s["positions"].long().reshape(-1)
  t, k = s["positions"].shape
  kept = (pos < s["offsets"][-1].long()).double()
  token = torch.arange(t, device=pos.device).repeat_interleave(k)
  rows = s["rows"].double()
  d = rows.shape[1]
  if kind == "from_experts_grad":
    dy = s["y_grad"].double()
    gain = s["weights"].double().reshape(-1) * kept
    drows = torch.zeros_like(rows).index_add_(
        0, pos, dy.index_select(0, token) * gain[:, None])
    dw = torch.einsum("nd,nd->n", rows.index_select(0, pos),
                      dy.index_select(0, token)) * kept
    return drows, dw.view(t, k)
  gain = kept
  if kind == "from_experts":
    gain = kept * s["weights"].double().reshape(-1)
  y = torch.zeros((t, d), dtype=torch.float64, device=pos.device)
  y.index_add_(0, token, rows.index_select(0, pos) * gain[:, None])
  return y


def _exact_adamw(s):
  f = lambda x: x.double().view(-1, BLOCK)
  g = f(s["g"]) * s["grad_scale"].double()
  if s["bits"] == 8:
    q = f(s["m"]) / 127
    m = q * q.abs() * s["m_scale"].double()
    v = ((f(s["v"]) / 255) ** 2 * s["v_scale"].double()) ** 2
  else:
    m, v = f(s["m"]), f(s["v"])
  t = s["step"] + 1
  m = torch.lerp(g, m, BETA_1)
  v = torch.lerp(g * g, v, BETA_2)
  mhat, vhat = m / (1 - BETA_1 ** t), v / (1 - BETA_2 ** t)
  p = f(s["p"])
  p = p - RATE * (mhat / (vhat.sqrt() + ADAM_EPSILON) +
                  DECAY * s["decays"].double() * p)
  out = {"p": p.view(-1)}
  if s["copies"] is not None:
    out["copies"] = p.view(-1)
  if s["bits"] == 8:
    top = m.abs().max(1, keepdim=True).values.clamp_min(1e-300)
    q = torch.round(127 * torch.sqrt(m.abs() / top))
    m = torch.sign(m) * top * (q / 127) ** 2
    r = v.sqrt()
    top = r.max(1, keepdim=True).values.clamp_min(1e-300)
    q = torch.round(255 * torch.sqrt(r / top))
    q[(q < 1) & (r > 0)] = 1
    v = (top * (q / 255) ** 2) ** 2
  out["m"], out["v"] = m.reshape(-1), v.reshape(-1)
  return out


def exact(case, seed):
  s = prepare(case, seed)
  if case["kind"].startswith("norm"):
    return _exact_norm(s, case["kind"] == "norm_grad")
  if case["kind"] == "adamw":
    return _exact_adamw(s)
  return _exact_experts(s)
