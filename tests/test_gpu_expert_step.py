"""The experts' products, the gradients' norm and what stands around them
together: a training step and scoring, eager, captured and on two streams."""

import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad  # pylint: disable=g-import-not-at-top,wrong-import-position

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.examples import ranking_moe  # pylint: disable=g-import-not-at-top,wrong-import-position
from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


class _Model:
  """Layer norm, a layer of experts and AdamW, with fixed inputs."""

  def __init__(self, seed, dtype, tokens=700, dim=96, hidden=104, experts=7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(s, device="cuda", generator=g)
    self.experts = experts
    self.x, self.target = new(tokens, dim).to(dtype), new(tokens, dim).to(dtype)
    self.ids = torch.randint(-1, experts, (tokens, 2), device="cuda",
                             generator=g)
    self.gates = torch.rand((tokens, 2), device="cuda", generator=g)
    self.up = (new(experts, dim, hidden) / dim**0.5).to(dtype)
    self.down = (new(experts, hidden, dim) / hidden**0.5).to(dtype)
    self.gain = torch.ones(dim, dtype=dtype, device="cuda")
    self.params = [self.up, self.down, self.gain]
    self.state = dense.init_adamw_state(self.params, state_bits=8)
    self.count = torch.zeros((), dtype=torch.int64, device="cuda")

  def forward(self):
    y, mean, rstd = dense.layer_norm(self.x, self.gain, return_stats=True)
    order = dense.sort_by_expert(self.ids, self.experts)
    rows = dense.tokens_to_experts(y, order)
    hidden = dense.expert_matmul(rows, self.up, order)
    active = torch.relu(hidden)
    out = dense.expert_matmul(active, self.down, order)
    return (dense.tokens_from_experts(out, self.gates, order), order, rows,
            hidden, active, out, mean, rstd)

  def step(self):
    self.count += 1
    y, order, rows, hidden, active, out, mean, rstd = self.forward()
    dout, _ = dense.tokens_from_experts_grad(y - self.target, out, self.gates,
                                             order)
    dactive, ddown = dense.expert_matmul_grad(dout, active, self.down, order)
    drows, dup = dense.expert_matmul_grad(dactive * (hidden > 0), rows, self.up,
                                          order)
    dy = dense.tokens_to_experts_grad(drows, order)
    _, dgain, _ = dense.layer_norm_grad(dy, self.x, mean, rstd, self.gain,
                                        with_bias=False)
    grads = [dup, ddown, dgain]
    norm, factor = dense.gradient_norm(grads, max_norm=1.0)
    dense.adamw_update(self.params, grads, self.state, learning_rate=0.01,
                       grad_scale=factor, step=self.count)
    clipped = [g.clone() for g in grads]
    again = dense.clip_gradients(clipped, 1.0)
    return [y, norm, factor, again, *grads, *clipped]

  def tensors(self):
    return [*self.params, self.state.m, self.state.v, self.state.m_scale,
            self.state.v_scale]


DTYPES = [torch.float32, torch.bfloat16]


def _same(a, b):
  for x, y in zip(a, b, strict=True):
    assert torch.equal(x, y)


def test_step_against_64_bits():
  m = _Model(0, torch.float32)
  p = [t.double().requires_grad_() for t in m.params]
  x = m.x.double()
  x = x - x.mean(1, keepdim=True)
  h = x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt() * p[2]
  y = 0
  for e in range(m.experts):
    gate = (m.gates.double() * (m.ids == e)).sum(1, keepdim=True)
    y = y + gate * (torch.relu(h @ p[0][e]) @ p[1][e])
  exact = torch.autograd.grad(((y - m.target.double())**2).sum() / 2, p)
  size = float(sum(g.square().sum() for g in exact)).__pow__(0.5)
  got = m.step()
  # float32 products over at most 700 values in half a dozen layers: 1e-4 of a
  # gradient's size is a hundred times their rounding.
  for g, e in zip(got[4:7], exact):
    assert float((g - e).norm()) <= 1e-4 * float(e.norm())
  assert abs(float(got[1]) - size) <= 1e-4 * size
  assert abs(float(got[2]) * size - 1) <= 1e-4
  assert float(got[3]) == float(got[1])
  total = sum(g.double().square().sum() for g in got[7:])
  assert abs(float(total) - 1) <= 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_step(dtype):
  """Each replay as the eager step, with eager work of the same operators and
  synchronizations in between."""
  eager, graphed, warm = (_Model(1, dtype) for _ in range(3))
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for _ in range(2):
      warm.step()
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = graphed.step()
  for _ in range(4):
    expected = eager.step()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    _same(out, expected)
    _same(graphed.tensors(), eager.tensors())
    warm.step()


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_streams(dtype):
  alone = [_Model(i, dtype, tokens=5000) for i in (1, 2)]
  expected = [[m.step() for _ in range(4)][-1] for m in alone]
  torch.cuda.synchronize()
  both = [_Model(i, dtype, tokens=5000) for i in (1, 2)]
  streams = [torch.cuda.Stream() for _ in both]
  torch.cuda.synchronize()
  outs = [None, None]
  for _ in range(4):
    for i, s in enumerate(streams):
      with torch.cuda.stream(s):
        outs[i] = both[i].step()
  torch.cuda.synchronize()
  for i in range(2):
    _same(outs[i], expected[i])
    _same(alone[i].tensors(), both[i].tensors())


def test_two_graphs_at_once():
  """Graphs captured one after another, replayed on two streams at once."""
  models = [_Model(i, torch.bfloat16, tokens=5000) for i in (1, 2)]
  queue = [dense.quantize_weights(m.up) for m in models]

  def work(m, q):
    order = dense.sort_by_expert(m.ids, m.experts)
    rows = dense.tokens_to_experts(m.x, order)
    return [dense.matmul_8bit(rows, q, order),
            *dense.expert_matmul_grad(rows, rows, m.up @ m.down, order),
            *dense.gradient_norm([m.x, m.up], max_norm=1.0)]

  expected = [work(m, q) for m, q in zip(models, queue)]
  torch.cuda.synchronize()
  graphs, outs = [], []
  for m, q in zip(models, queue):
    graphs.append(torch.cuda.CUDAGraph())
    with torch.cuda.graph(graphs[-1]):
      outs.append(work(m, q))
  streams = [torch.cuda.Stream() for _ in models]
  for _ in range(4):
    for out in outs:
      for t in out:
        t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
      for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
          graph.replay()
    torch.cuda.synchronize()
    for out, e in zip(outs, expected):
      _same(out, e)


def test_example_scores_in_8_bits():
  config = ranking_moe.Config(batch=256, vocabulary=500, max_norm=0.1)
  model = ranking_moe.RankingModel(config)
  ids, clicks = ranking_moe.Clicks(config).batch()
  model.step(ids, clicks)
  experts = model.quantize_experts()
  plain, scored = model.score(ids), model.score(ids, experts)
  assert scored.shape == plain.shape == (256,)
  # With the weights that the codes stand for the products are the same but for
  # the rows' rounding: the same call with its parts by hand.
  _, acts = model.lookup(ids)
  with torch.no_grad():
    w = model.weights
    x = dense.layer_norm(torch.cat(acts, 1), w["norm_in"], w["norm_in_bias"])
    top, chosen = (x @ w["router"]).topk(config.choices, dim=1)
    order = dense.sort_by_expert(chosen, config.experts)
    rows = dense.tokens_to_experts(x, order)
    rows = torch.relu(dense.matmul_8bit(rows, experts["up"], order))
    rows = dense.matmul_8bit(rows, experts["down"], order)
    y = dense.tokens_from_experts(rows, top.softmax(1), order)
    y = dense.layer_norm(x + y, w["norm_out"], w["norm_out_bias"])
    assert torch.equal(scored, (y @ w["logit"]).squeeze(1).sigmoid())


def test_example_clips():
  """Gradients far below the limit: the step without clipping."""
  config = ranking_moe.Config(batch=128, vocabulary=300)
  runs = []
  for limit in (None, 1e6):
    c = ranking_moe.Config(batch=128, vocabulary=300, max_norm=limit)
    model, clicks = ranking_moe.RankingModel(c), ranking_moe.Clicks(config)
    for _ in range(3):
      model.step(*clicks.batch())
    runs.append([p.detach() for p in model.weights.values()])
  _same(*runs)


@pytest.mark.parametrize("name", ["rows", "weights", "y_grad", "rows_8",
                                  "quantize", "norm", "clip"])
def test_a_tangent_is_refused(name):
  x, w = torch.ones((6, 8), device="cuda"), torch.ones((2, 8, 8),
                                                       device="cuda")
  order = dense.sort_by_expert(torch.tensor([0, 1, 0, 1, 0, 0],
                                            device="cuda"), 2)
  q = dense.quantize_weights(w)
  call, t = {
      "rows": (lambda t: dense.expert_matmul(t, w, order), x),
      "weights": (lambda t: dense.expert_matmul(x, t, order), w),
      "y_grad": (lambda t: dense.expert_matmul_grad(t, x, w, order), x),
      "rows_8": (lambda t: dense.matmul_8bit(t, q, order), x),
      "quantize": (dense.quantize_weights, w),
      "norm": (lambda t: dense.gradient_norm([t]), x),
      "clip": (lambda t: dense.clip_gradients([t], 1.0), x),
  }[name]
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(t, torch.ones_like(t))
    with pytest.raises(ValueError, match="tangent"):
      call(dual)
    call(t)


def test_values_that_are_not_in_memory():
  x, w = torch.randn((9, 24), device="cuda"), torch.randn((2, 24, 16),
                                                          device="cuda")
  dy = torch.randn((9, 16), device="cuda")
  order = dense.sort_by_expert(torch.arange(9, device="cuda") % 2, 2)
  neg = torch._neg_view  # pylint: disable=protected-access
  assert torch.equal(dense.expert_matmul(neg(-x), neg(-w), order),
                     dense.expert_matmul(x, w, order))
  _same(dense.expert_matmul_grad(neg(-dy), neg(-x), neg(-w), order),
        dense.expert_matmul_grad(dy, x, w, order))
  _same(dense.quantize_weights(neg(-w))[1:2], dense.quantize_weights(w)[1:2])


@pytest.fixture
def _small_memory():
  torch.cuda.empty_cache()
  total = torch.cuda.get_device_properties(0).total_memory
  most = torch.cuda.memory_reserved() + (1 << 30)
  torch.cuda.set_per_process_memory_fraction(most / total)
  yield
  torch.cuda.set_per_process_memory_fraction(1.0)


def test_out_of_memory_is_torchs(_small_memory):
  x = torch.ones((1, 8), device="cuda").expand(1 << 20, 8)
  w = torch.ones((1, 8, 1), device="cuda").expand(1, 8, 1 << 14)
  order = dense.ExpertOrder(None, None, torch.tensor(
      [0, 1 << 20], dtype=torch.int32, device="cuda"))
  for call in (lambda: dense.expert_matmul(x, w, order),
               lambda: dense.gradient_norm([x.expand(1 << 10, -1, -1)])):
    with pytest.raises(torch.OutOfMemoryError):
      call()
  assert dense.expert_matmul(x[:3], w[:, :, :5], order).shape == (3, 5)
