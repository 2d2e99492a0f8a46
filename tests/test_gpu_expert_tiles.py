"""The experts' products (lib/nn/dense.py) by each size of tile and way of loading
that large calls take, bit for bit: whole numbers, whose sums are exact in float32
and rounded once.

A launch has tiles of 256 x 256 where 256 CUs have at least four fifths of their
last round, and of 128 x 128 where those are fewer; the sizes here are far from
both borders (500 tiles of 256 x 256; 240 or more of 128 x 128 and a result one
large tile wide).
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


def _whole(shape, dtype, seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  return torch.randint(-3, 4, shape, device="cuda", generator=g).to(dtype)


def _offsets(counts):
  out = [0]
  for c in counts:
    out.append(out[-1] + c)
  return out


def _run(counts, inner, outer, stored, dtype, dropped=5, weights_only=False):
  offsets = _offsets(counts)
  n, experts = offsets[-1] + dropped, len(counts)
  x, dy = _whole((n, inner), dtype, 1), _whole((n, outer), dtype, 2)
  w = _whole((experts, inner, outer), dtype, 3)
  if stored == "out_in":
    w = w.transpose(1, 2).contiguous().transpose(1, 2)
  x[offsets[-1]:] = float("nan")
  dy[offsets[-1]:] = float("inf")
  order = dense.ExpertOrder(None, None, torch.tensor(
      offsets, dtype=torch.int32, device="cuda"))
  y = None if weights_only else dense.expert_matmul(x, w, order)
  dx, dw = dense.expert_matmul_grad(dy, x, w, order,
                                    with_rows=not weights_only)
  for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
    xe, we, ge = x[a:b].double(), w[e].double(), dy[a:b].double()
    assert torch.equal(dw[e], torch.mm(xe.t().contiguous(), ge).to(dtype)), e
    if not weights_only:
      assert torch.equal(y[a:b], torch.mm(xe, we.contiguous()).to(dtype)), e
      assert torch.equal(dx[a:b], torch.mm(
          ge, we.t().contiguous()).to(dtype)), e
  if not weights_only:
    assert not y[offsets[-1]:].any() and not dx[offsets[-1]:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stored", ["in_out", "out_in"])
@pytest.mark.parametrize("counts", [
    [32_000], [7000, 0, 13_777, 1, 11_215], [1900] * 17])
def test_large_tiles(counts, stored, dtype):
  """500 tiles of 256 x 256 in both directions (float32: four times as many of
  128 x 128); with 17 experts the weights' gradient has 272 of them too, ranked
  by length, all equal."""
  _run(counts, 776, 776, stored, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stored", ["in_out", "out_in"])
@pytest.mark.parametrize("inner,outer", [(100, 131), (131, 100), (104, 136),
                                         (257, 129)])
def test_middle_tiles(inner, outer, stored, dtype):
  """235 rows of tiles of 128 x 128; rows that are whole 16 bytes, that are not,
  and (100 float32 values) that are beside weights that are not."""
  _run([9000, 0, 20_001, 1000], inner, outer, stored, dtype)


def _ragged(experts, each):
  """Counts around `each`, some equal, some none, one very long, and whole
  numbers of steps of 32 and 64 rows among them, even and odd."""
  some = [each, each + 64, each, 0, each - 1, 64, each + 32, 1, 2 * each + 96,
          each + 1]
  counts = [some[i % len(some)] for i in range(experts)]
  counts[experts // 2] = 5 * each
  short = 256 * experts - sum(counts)
  counts[0] += max(short, 0)
  return counts


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stored", ["in_out", "out_in"])
@pytest.mark.parametrize("experts", [64, 65, 200, 256, 257])
def test_weights_of_many_experts(experts, stored, dtype):
  """The weights' gradient by tiles of 256 x 256 (float32: 128 x 128), of whole
  steps and remainders, experts in the order of their lengths up to 256 of
  them."""
  _run(_ragged(experts, 320), 264, 520, stored, dtype, weights_only=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stored", ["in_out", "out_in"])
def test_odd_weights_of_many_experts(stored, dtype):
  """The same through registers."""
  _run(_ragged(65, 320), 259, 515, stored, dtype, weights_only=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_few_rows_of_many_experts(dtype):
  """Below 256 rows an expert: in their own order."""
  _run([(i * 37) % 300 for i in range(100)], 264, 520, "in_out", dtype,
       weights_only=True)
