"""Captured calls and their scratch memory: graphs that were captured one after
another on the same stream (torch's default capture stream) may be replayed at
once, and beside eager work."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore import _native  # pylint: disable=g-import-not-at-top,wrong-import-position
from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _span(buf):
  return buf.data_ptr(), buf.data_ptr() + buf.numel()


def test_captured_scratch_is_the_graphs_own():
  """No graph's scratch overlaps another's, or that of eager calls on the
  stream that it was captured on."""
  stream = torch.cuda.Stream()
  spans, graphs = [], []
  with torch.cuda.stream(stream):
    spans.append(_span(_native.WORKSPACE.get(1 << 16)))
  for _ in range(2):
    graphs.append(torch.cuda.CUDAGraph())
    x = torch.zeros(8, device="cuda")
    with torch.cuda.graph(graphs[-1], stream=stream):
      x.add_(1)
      spans.append(_span(_native.WORKSPACE.get(1 << 16)))
  # A stream that is given, forked from the capture.
  side = torch.cuda.Stream()
  graphs.append(torch.cuda.CUDAGraph())
  with torch.cuda.graph(graphs[-1], stream=stream):
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      x.add_(1)
    spans.append(_span(_native.WORKSPACE.get(1 << 16, side)))
    torch.cuda.current_stream().wait_stream(side)
  with torch.cuda.stream(stream):
    assert _span(_native.WORKSPACE.get(1 << 16)) == spans[0]
  spans.sort()
  for (_, end), (begin, _) in zip(spans, spans[1:]):
    assert end <= begin


def test_graphs_at_once():
  """Two graphs of sorts (in tiles, with a workspace) and layer norm's gradient,
  replayed on two streams beside an eager pass on a third."""
  tokens, dim, experts = 30_000, 264, 40

  def make(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((tokens, dim), device="cuda", generator=g)
    ids = torch.randint(-1, experts, (tokens, 2), device="cuda", generator=g)
    return x, ids, torch.rand(dim, device="cuda", generator=g)

  def step(x, ids, w):
    order = dense.sort_by_expert(ids, experts)
    y, mean, rstd = dense.layer_norm(x, w, return_stats=True)
    return (*order, *dense.layer_norm_grad(y, x, mean, rstd, w))

  data = [make(seed) for seed in (1, 2, 3)]
  expected = [step(*d) for d in data]
  graphs, outs = [], []
  torch.cuda.synchronize()
  for d in data[:2]:
    graphs.append(torch.cuda.CUDAGraph())
    with torch.cuda.graph(graphs[-1]):
      outs.append(step(*d))
  streams = [torch.cuda.Stream() for _ in data]
  for _ in range(5):
    for out in outs:
      for t in out:
        t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
      for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
          graph.replay()
      with torch.cuda.stream(streams[2]):
        eager = step(*data[2])
    torch.cuda.synchronize()
    for got, want in zip([*outs, eager], expected):
      for a, b in zip(got, want, strict=True):
        assert torch.equal(a, b)
