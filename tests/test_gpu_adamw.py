"""AdamW over many tensors (lib/nn/dense.py).

float32 moments and the weights are held against the definition in 64 bits: u
being float32's unit roundoff, a new moment is off by at most 4 u of the
magnitudes that it is the sum of, the update m / (sqrt(v) / sqrt(c) + eps) by
16 u of itself beside what m's error brings, the weight by its own rounding and
2 u of itself.

Moments of 8 bits are held bit for bit against the same steps in numpy's
float32, whose products, sums, quotients and roots are correctly rounded, and
the codes' meaning (nearest code, no zero for a second moment above zero)
against 64 bits.
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

U = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
HYPER = dict(learning_rate=0.01, beta_1=0.9, beta_2=0.99, epsilon=1e-7,
             weight_decay=0.1)
SIZES = [1, 3, 0, 4, 255, 256, 257, 1000, 1024, 4095, 4096, 4097, 20011]
F = np.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _tensors(sizes, dtype, seed, scale=1.0, offset=0):
  """Tensors of the sizes; offset: values before the first, which shifts them
  off 16 bytes."""
  g = torch.Generator(device="cuda").manual_seed(seed)
  out = []
  for n in sizes:
    x = torch.randn(n + offset, device="cuda", generator=g) * scale
    out.append(x.to(dtype)[offset:])
  return out


class _Exact:
  """The definition in 64 bits, one tensor."""

  def __init__(self, p, decay=True):
    self.p = p.double().cpu().numpy()
    self.m = np.zeros_like(self.p)
    self.v = np.zeros_like(self.p)
    self.t = 0
    self.decay = decay

  def step(self, g, learning_rate, beta_1, beta_2, epsilon, weight_decay,
           scale=1.0):
    """Returns tolerances (of p without its own rounding, of m, of v)."""
    self.t += 1
    g = g.double().cpu().numpy() * scale
    mm = beta_1 * np.abs(self.m) + (1 - beta_1) * np.abs(g)
    self.m = beta_1 * self.m + (1 - beta_1) * g
    self.v = beta_2 * self.v + (1 - beta_2) * g * g
    denom = np.sqrt(self.v) / math.sqrt(1 - beta_2 ** self.t) + epsilon
    rate = learning_rate / (1 - beta_1 ** self.t)
    keep = 1 - (learning_rate * weight_decay if self.decay else 0.0)
    self.p = self.p * keep - rate * self.m / denom
    return (2 * U * np.abs(self.p) + rate * (
        16 * U * np.abs(self.m) + 4 * U * mm) / denom, 4 * U * mm,
            6 * U * self.v)


def _cpu(x):
  return x.detach().double().cpu().numpy()


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32),
                                   (torch.float32, torch.bfloat16),
                                   (torch.bfloat16, torch.bfloat16),
                                   (torch.bfloat16, torch.float32)], ids=str)
def test_float32_moments(types, offset):
  """Each step from the state that the last one left."""
  ptype, gtype = types
  params = _tensors(SIZES, ptype, 1, offset=offset)
  decay = [i % 3 != 0 for i in range(len(SIZES))]
  state = dense.init_adamw_state(params, decay=decay)
  copies = [torch.zeros(n + offset, dtype=torch.bfloat16,
                        device="cuda")[offset:] for n in SIZES]
  for t in range(3):
    exact = [_Exact(p, d) for p, d in zip(params, decay)]
    for e, at, n in zip(exact, state.first, SIZES):
      e.m, e.v = _cpu(state.m[at:at + n]), _cpu(state.v[at:at + n])
      e.t = t
    grads = _tensors(SIZES, gtype, 10 + t, offset=offset)
    got = dense.adamw_update(params, grads, state, copies=copies, **HYPER)
    assert state.step == t + 1
    for i, (e, at, n) in enumerate(zip(exact, state.first, SIZES)):
      ptol, mtol, vtol = e.step(grads[i], **HYPER)
      assert got[i] is params[i]
      assert (np.abs(_cpu(params[i]) - e.p) <= ptol +
              ROUND[ptype] * np.abs(e.p) * (1 + 1e-3)).all(), (t, n)
      assert (np.abs(_cpu(state.m[at:at + n]) - e.m) <= mtol + 1e-37).all()
      assert (np.abs(_cpu(state.v[at:at + n]) - e.v) <= vtol + 1e-37).all()
      if ptype == torch.bfloat16:
        assert torch.equal(copies[i], params[i])
      else:
        assert torch.equal(copies[i], params[i].bfloat16())
  m, v = dense.adamw_moments(state)
  assert m is state.m and v is state.v
  used = torch.zeros_like(m, dtype=torch.bool)
  for at, n in zip(state.first, SIZES):
    used[at:at + n] = True
  assert (m[~used] == 0).all() and (v[~used] == 0).all()


def _encode_m(m):
  s = np.abs(m).max()
  if s == 0:
    return np.zeros(m.shape, np.int8), s
  q = np.rint(np.sqrt(np.abs(m) / s) * F(127))
  return np.where(m < 0, -q, q).astype(np.int8), s


def _encode_r(r):
  s = r.max()
  if s == 0:
    return np.zeros(r.shape, np.uint8), s
  q = np.rint(np.sqrt(r / s) * F(255))
  return np.maximum(q, (r > 0).astype(F)).astype(np.uint8), s


def _blocks(x):
  n = -(-x.size // 256) * 256
  out = np.zeros(n, x.dtype)
  out[:x.size] = x
  return out.reshape(-1, 256)


@pytest.mark.parametrize("offset,size", [(0, 1.0), (1, 1.0), (0, 1e-33),
                                         (0, 1e-18), (0, 1e-12), (0, 1e-6),
                                         (0, 1e9), (0, 1e17)])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16], ids=str)
def test_8_bit_moments(gtype, offset, size):
  """size: of the gradients; second moments from none (they underflow) to near
  the largest float32."""
  params = _tensors(SIZES, torch.float32, 2, offset=offset)
  state = dense.init_adamw_state(params, state_bits=8)
  host = [(np.zeros(n, F), np.zeros(n, F)) for n in SIZES]  # m, root of v
  for t in range(1, 5):
    # Blocks of very different gradients, zeros among them.
    grads = _tensors(SIZES, gtype, 20 + t, offset=offset)
    for g in grads:
      g *= torch.exp(3 * torch.sin(torch.arange(g.numel(), device="cuda"))).to(
          gtype)
      g[g.abs() < 0.05] = 0
      g *= size
    before = [_cpu(p).astype(F) for p in params]
    dense.adamw_update(params, grads, state, grad_scale=0.5, **HYPER)
    for i, n in enumerate(SIZES):
      g = _cpu(grads[i]).astype(F) * F(0.5)
      m, r = host[i]
      m = m * F(0.9) + g * F(1 - 0.9)
      v = r * r
      v = v * F(0.99) + g * g * F(1 - 0.99)
      r = np.sqrt(v)
      root = F(1 / math.sqrt(1 - 0.99 ** t))
      p = before[i] * F(1 - 0.001) - m / (r * root + F(1e-7)) * F(
          0.01 / (1 - 0.9 ** t))
      assert (np.abs(_cpu(params[i]) - p) <= 4 * U * np.abs(p) + 32 * U *
              0.01 * np.abs(m / (r * root + F(1e-7)))).all()
      at = state.first[i]
      qm, qv = (_blocks(x.cpu().numpy()[at:at + n]) for x in (state.m, state.v))
      ms, vs = (x.cpu().numpy()[at // 256:-(-(at + n) // 256)]
                for x in (state.m_scale, state.v_scale))
      nm, nr = [], []
      for b, (bm, br) in enumerate(zip(_blocks(m), _blocks(r))):
        em, es = _encode_m(bm)
        er, eq = _encode_r(br)
        assert ms[b] == es and vs[b] == eq, (t, n, b)
        assert np.array_equal(qm[b], em) and np.array_equal(qv[b], er)
        # What the codes mean, in 64 bits.
        if es > 0:
          x = np.sign(bm) * np.sqrt(np.abs(bm.astype(np.float64)) / es) * 127
          assert np.abs(x - qm[b]).max() <= 0.5 + 1e-4
        assert ((br > 0) == (qv[b] > 0)).all()
        x = em.astype(F) * F(1 / 127)
        nm.append(x * np.abs(x) * es)
        x = er.astype(F) * F(1 / 255)
        nr.append(x * x * eq)
      host[i] = (np.concatenate(nm)[:n] if nm else m,
                 np.concatenate(nr)[:n] if nr else r)
  m, v = dense.adamw_moments(state)
  for i, n in enumerate(SIZES):
    at = state.first[i]
    assert np.array_equal(m[at:at + n].cpu().numpy(), host[i][0])
    assert np.array_equal(v[at:at + n].cpu().numpy(), host[i][1] * host[i][1])


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors(bits):
  """More tensors than one launch takes, some without a gradient; the same as
  one tensor at a time."""
  sizes = [(7 * i) % 613 + 1 for i in range(150)]
  grads = _tensors(sizes, torch.float32, 5)
  for i in (0, 3, 64, 149):
    grads[i] = None
  together = _tensors(sizes, torch.float32, 6)
  alone = [p.clone() for p in together]
  state = dense.init_adamw_state(together, state_bits=bits)
  states = [dense.init_adamw_state([p], state_bits=bits) for p in alone]
  for _ in range(2):
    dense.adamw_update(together, grads, state, **HYPER)
    for p, g, s in zip(alone, grads, states):
      dense.adamw_update([p], [g], s, **HYPER)
  m, v = dense.adamw_moments(state)
  for i, (p, q) in enumerate(zip(together, alone)):
    assert torch.equal(p, q)
    at, n = state.first[i], sizes[i]
    sm, sv = dense.adamw_moments(states[i])
    assert torch.equal(m[at:at + n], sm[:n]) and torch.equal(v[at:at + n],
                                                             sv[:n])
    if grads[i] is None:
      assert (m[at:at + n] == 0).all()
  assert torch.equal(together[0], _tensors(sizes, torch.float32, 6)[0])


@pytest.mark.parametrize("count", [63, 64, 65, 83, 84, 87, 88, 104, 105, 108,
                                   109, 129, 217])
def test_numbers_of_tensors(count):
  """On both sides of what a launch and a lane take, with and without copies,
  against one tensor that holds them all."""
  sizes = [256 * (1 + i % 5) for i in range(count)]
  for with_copies in (False, True):
    flat, grad = _tensors([sum(sizes)], torch.float32, 1)[0], _tensors(
        [sum(sizes)], torch.bfloat16, 2)[0]
    other = flat.clone()
    copy = torch.zeros_like(grad)
    params, grads, copies = (list(x.split(sizes)) for x in (flat, grad, copy))
    if with_copies:
      copies[count // 2] = None
    state = dense.init_adamw_state(params, state_bits=8)
    one = dense.init_adamw_state([other], state_bits=8)
    dense.adamw_update(params, grads, state, **HYPER,
                       copies=copies if with_copies else None)
    dense.adamw_update([other], [grad], one, **HYPER)
    assert torch.equal(flat, other)
    for name in ("m", "v", "m_scale", "v_scale"):
      assert torch.equal(getattr(state, name), getattr(one, name))
    for i, c in enumerate(copy.split(sizes)):
      written = with_copies and i != count // 2
      assert torch.equal(c, params[i].bfloat16() if written else
                         torch.zeros_like(c))


@pytest.mark.parametrize("bits", [8, 32])
def test_hyperparameters_on_the_gpu(bits):
  """Device scalars give what host values give; their factors are made in 64
  bits on either side, so the weights agree to a rounding."""
  sizes = [5000, 77]
  params = _tensors(sizes, torch.float32, 1)
  other = [p.clone() for p in params]
  a = dense.init_adamw_state(params, state_bits=bits)
  b = dense.init_adamw_state(other, state_bits=bits)
  rate = torch.tensor(0.01, device="cuda")
  scale = torch.tensor([0.25], device="cuda")
  step = torch.zeros((), dtype=torch.int64, device="cuda")
  hyper = {**HYPER, "learning_rate": float(rate)}
  for t in range(3):
    grads = _tensors(sizes, torch.float32, 30 + t)
    dense.adamw_update(params, grads, a, grad_scale=0.25, **hyper)
    step += 1
    dense.adamw_update(other, grads, b, grad_scale=scale, step=step,
                       **{**hyper, "learning_rate": rate})
    for p, q in zip(params, other):
      assert ((p - q).abs() <= 8 * U * (p.abs() + 0.1)).all()
    assert torch.equal(a.m, b.m) and torch.equal(a.v, b.v)
  assert a.step == 3 and b.step == 0
  dense.adamw_update(params, grads, a, step=10, **hyper)
  assert a.step == 10


def test_no_epsilon_and_no_gradient_yet():
  """A value that never had a gradient: 0 / (0 + epsilon) is zero."""
  for bits in (8, 32):
    p = torch.ones(300, device="cuda")
    g = torch.zeros(300, device="cuda")
    g[:10] = 1.0
    state = dense.init_adamw_state([p], state_bits=bits)
    dense.adamw_update([p], [g], state, learning_rate=0.1, weight_decay=0.0)
    assert (p[10:] == 1).all() and (p[:10] < 0.91).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_not_finite_gradients(bits):
  """They reach their own values, with 8 bits their block's moments, and no
  other block."""
  p = torch.ones(1024, device="cuda")
  g = torch.full((1024,), 0.5, device="cuda")
  g[300], g[301] = float("nan"), float("inf")
  state = dense.init_adamw_state([p], state_bits=bits)
  dense.adamw_update([p], [g], state, **HYPER)
  bad = torch.zeros(1024, dtype=torch.bool, device="cuda")
  bad[300] = bad[301] = True
  assert p[~bad].isfinite().all() and p[bad].isnan().all()
  m, v = dense.adamw_moments(state)
  if bits == 8:
    bad[256:512] = True
    assert m[bad].isnan().all()
  assert m[~bad].isfinite().all() and v[~bad].isfinite().all()
  assert not m[300].isfinite() and not v[301].isfinite()


@pytest.mark.parametrize("types", [(torch.float32, torch.float32),
                                   (torch.float32, torch.bfloat16),
                                   (torch.bfloat16, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("bits", [8, 32])
def test_more_than_the_caches(bits, types):
  """Steps of more than 256 MB go past the caches: the same bits as in parts."""
  ptype, gtype = types
  n, parts = 64_000_513, 8
  p = _tensors([n], ptype, 1)[0]
  g = _tensors([n], gtype, 2)[0]
  step = 8_000_000
  assert step % 256 == 0 and step * parts < n
  q = p.clone()
  cuts = [slice(i * step, (i + 1) * step if i < parts else n)
          for i in range(parts + 1)]
  copy = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
  whole = dense.init_adamw_state([p], state_bits=bits)
  states = [dense.init_adamw_state([q[c]], state_bits=bits) for c in cuts]
  for _ in range(2):
    dense.adamw_update([p], [g], whole, copies=[copy], **HYPER)
    for c, s in zip(cuts, states):
      dense.adamw_update([q[c]], [g[c]], s, **HYPER)
  assert torch.equal(p, q) and torch.equal(copy, p.bfloat16())
  for name in ("m", "v") + (("m_scale", "v_scale") if bits == 8 else ()):
    assert torch.equal(getattr(whole, name),
                       torch.cat([getattr(s, name) for s in states])), name


def test_large_tensor():
  """More than 2^31 bytes in one tensor, checked at both ends."""
  n = 600_000_007
  p = torch.zeros(n, device="cuda")
  g = torch.ones(n, dtype=torch.bfloat16, device="cuda")
  state = dense.init_adamw_state([p], state_bits=8)
  dense.adamw_update([p], [g], state, learning_rate=0.5, weight_decay=0.0)
  assert (p[:5000] + 0.5).abs().max() < 1e-5
  assert (p[-5000:] + 0.5).abs().max() < 1e-5
  assert int(state.m[n - 1]) == 127 and int(state.v[n - 1]) == 255


def test_refusals():
  p = torch.ones(64, device="cuda")
  g = torch.ones(64, device="cuda")
  state = dense.init_adamw_state([p])
  before = p.clone()
  up = lambda ps, gs, s=state, **k: dense.adamw_update(
      ps, gs, s, **{**HYPER, **k})
  bad = [
      lambda: dense.init_adamw_state([p], state_bits=16),
      lambda: dense.init_adamw_state([p.double()]),
      lambda: dense.init_adamw_state([p.cpu()]),
      lambda: dense.init_adamw_state([p.view(8, 8).t()]),
      lambda: dense.init_adamw_state([p], decay=[True, False]),
      lambda: up([p, p], [g, g]),
      lambda: up([p, p], [g, g], dense.init_adamw_state([p, p])),
      lambda: up([p[:40], p[32:]], [g[:40], g[32:]],
                 dense.init_adamw_state([p[:40], p[32:]])),
      lambda: up([p], [g, g]),
      lambda: up([p], [g[:8]]),
      lambda: up([p], [g.double()]),
      lambda: up([p], [g.cpu()]),
      lambda: up([p[:8]], [g[:8]]),
      lambda: up([p], [g], copies=[p]),
      lambda: up([p], [g], copies=[]),
      lambda: up([p], [g], copies=[p.bfloat16()[:8]]),
      lambda: up([p], [g], beta_1=1.0),
      lambda: up([p], [g], beta_2=-0.1),
      lambda: up([p], [g], epsilon=-1e-8),
      lambda: up([p], [g], step=0),
      lambda: up([p], [g], learning_rate=torch.ones(2, device="cuda")),
  ]
  for i, call in enumerate(bad):
    with pytest.raises(ValueError):
      call()
      print("not refused:", i)
  assert torch.equal(p, before) and state.step == 0


def test_strided_gradients_and_shapes():
  p = torch.randn((30, 40), device="cuda")
  q = p.clone()
  g = torch.randn((40, 30), device="cuda").t()
  a, b = dense.init_adamw_state([p]), dense.init_adamw_state([q])
  dense.adamw_update([p], [g], a, **HYPER)
  dense.adamw_update([q], [g.contiguous()], b, **HYPER)
  assert torch.equal(p, q)
  one = torch.ones((), device="cuda").expand(30, 40)
  dense.adamw_update([p], [one], a, **HYPER)
  dense.adamw_update([q], [torch.ones_like(q)], b, **HYPER)
  assert torch.equal(p, q)
  dense.adamw_update([], [], dense.init_adamw_state([]), **HYPER)
