"""The dense operators together: the example's training step against the same
model in 64 bits, and a captured step replayed."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.examples import ranking_moe  # pylint: disable=g-import-not-at-top,wrong-import-position
from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _plain_loss(config, weights, acts, clicks, ids):
  """The example's model in the tensors' own precision, every expert on every
  sample; `ids` are the experts that the router chose."""
  def norm(x, w, b):
    x = x - x.mean(1, keepdim=True)
    return x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt() * w + b

  x = norm(torch.cat(acts, 1), weights["norm_in"], weights["norm_in_bias"])
  scores = (x @ weights["router"]).gather(1, ids).softmax(1)
  y = 0
  for e in range(config.experts):
    gate = (scores * (ids == e)).sum(1, keepdim=True)
    y = y + gate * (torch.relu(x @ weights["up"][e]) @ weights["down"][e])
  y = norm(x + y, weights["norm_out"], weights["norm_out_bias"])
  return torch.nn.functional.binary_cross_entropy_with_logits(
      (y @ weights["logit"]).squeeze(1), clicks)


@pytest.mark.parametrize("choices", [1, 3])
def test_example_gradients(choices):
  config = ranking_moe.Config(batch=256, choices=choices, vocabulary=500)
  model = ranking_moe.RankingModel(config)
  ids, clicks = ranking_moe.Clicks(config).batch()
  _, acts = model.lookup(ids)
  params = list(model.weights.values())
  loss = torch.nn.functional.binary_cross_entropy_with_logits(
      model.logits(acts), clicks)
  grads = torch.autograd.grad(loss, acts + params)
  w = {k: v.detach().double().requires_grad_()
       for k, v in model.weights.items()}
  a = [x.detach().double().requires_grad_() for x in acts]
  x = dense.layer_norm(torch.cat(acts, 1), model.weights["norm_in"],
                       model.weights["norm_in_bias"])
  chosen = (x @ model.weights["router"]).topk(choices, dim=1).indices
  exact = _plain_loss(config, w, a, clicks.double(), chosen)
  expected = torch.autograd.grad(exact, a + list(w.values()))
  # float32 products over at most 256 values in a dozen layers, forwards and
  # back: 1e-4 of a gradient's size is a hundred times their rounding.
  assert abs(loss.item() - exact.item()) < 1e-5
  for g, e in zip(grads, expected):
    assert float((g - e).norm()) <= 1e-4 * float(e.norm()) + 1e-9


@pytest.mark.parametrize("bits", [8, 32])
def test_example_learns(bits):
  """The clicks are a function of the ids: the loss of a balanced coin, ln 2,
  falls."""
  losses = ranking_moe.train(
      ranking_moe.Config(state_bits=bits, vocabulary=1000), 60)
  assert np.isfinite(losses).all()
  assert np.mean(losses[-10:]) < 0.9 * np.mean(losses[:3])


def test_two_streams():
  """Steps on two streams at once, each with its own data and workspace."""
  tokens, dim, experts = 20_000, 264, 40

  def make(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((tokens, dim), device="cuda", generator=g)
    ids = torch.randint(-1, experts, (tokens, 2), device="cuda", generator=g)
    gates = torch.rand((tokens, 2), device="cuda", generator=g)
    p = [torch.ones(dim, device="cuda"), torch.zeros(dim, device="cuda")]
    return x, ids, gates, p, dense.init_adamw_state(p, state_bits=8)

  def step(x, ids, gates, p, state):
    y, mean, rstd = dense.layer_norm(x, *p, return_stats=True)
    order = dense.sort_by_expert(ids, experts)
    rows = dense.tokens_to_experts(y, order)
    out = dense.tokens_from_experts(rows, gates, order)
    drows, _ = dense.tokens_from_experts_grad(out, rows, gates, order)
    dy = dense.tokens_to_experts_grad(drows, order)
    _, dw, db = dense.layer_norm_grad(dy, x, mean, rstd, p[0])
    dense.adamw_update(p, [dw, db], state, learning_rate=0.01)
    return out

  alone = [make(i) for i in (1, 2)]
  expected = [[step(*a) for _ in range(5)][-1] for a in alone]
  torch.cuda.synchronize()
  both = [make(i) for i in (1, 2)]
  streams = [torch.cuda.Stream() for _ in both]
  torch.cuda.synchronize()
  outs = [None, None]
  for _ in range(5):
    for i, s in enumerate(streams):
      with torch.cuda.stream(s):
        outs[i] = step(*both[i])
  torch.cuda.synchronize()
  for i in range(2):
    assert torch.equal(outs[i], expected[i])
    for a, b in zip(alone[i][3], both[i][3]):
      assert torch.equal(a, b)
    assert torch.equal(alone[i][4].m, both[i][4].m)


def test_captured_step():
  """Norm, experts and AdamW with a step counter on the GPU, captured once and
  replayed with other work in between: each replay as the eager step."""
  tokens, dim, experts = 300, 96, 5
  g = torch.Generator(device="cuda").manual_seed(0)
  new = lambda *s: torch.randn(s, device="cuda", generator=g)
  x, target = new(tokens, dim), new(tokens, dim)
  ids = torch.randint(-1, experts, (tokens, 2), device="cuda", generator=g)
  gates = torch.rand((tokens, 2), device="cuda", generator=g)

  def make():
    gg = torch.Generator(device="cuda").manual_seed(1)
    p = [1 + 0.1 * torch.randn(dim, device="cuda", generator=gg),
         0.1 * torch.randn(dim, device="cuda", generator=gg)]
    return p, dense.init_adamw_state(p, state_bits=8), torch.zeros(
        (), dtype=torch.int64, device="cuda")

  def step(p, state, count):
    count += 1
    y, mean, rstd = dense.layer_norm(x, p[0], p[1], return_stats=True)
    order = dense.sort_by_expert(ids, experts)
    rows = dense.tokens_to_experts(y, order)
    out = dense.tokens_from_experts(rows, gates, order)
    drows, _ = dense.tokens_from_experts_grad(out - target, rows, gates, order)
    dy = dense.tokens_to_experts_grad(drows, order)
    _, dw, db = dense.layer_norm_grad(dy, x, mean, rstd, p[0])
    dense.adamw_update(p, [dw, db], state, learning_rate=0.01, step=count)
    return out

  eager, graphed = make(), make()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    warm = make()
    for _ in range(2):
      step(*warm)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step(*graphed)
  for _ in range(4):
    expected = step(*eager)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, expected)
    assert int(graphed[2]) == int(eager[2])
    for a, b in zip(graphed[0], eager[0]):
      assert torch.equal(a, b)
    for name in ("m", "v", "m_scale", "v_scale"):
      assert torch.equal(getattr(graphed[1], name), getattr(eager[1], name))
    new(1000, 1000).sum().item()
