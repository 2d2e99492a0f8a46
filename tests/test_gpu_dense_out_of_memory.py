"""Running out of GPU memory in a dense operator is torch's own error, which
callers catch to free memory and try again. The allocator's own limit is set
low, so it refuses before it asks the device."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from jax_tpu_embedding.sparsecore.lib.nn import dense  # pylint: disable=g-import-not-at-top,wrong-import-position


@pytest.fixture(scope="module", autouse=True)
def _gpu():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  torch.cuda.set_device(0)


@pytest.fixture
def small_memory():
  """A limit of about 1 GiB above what is reserved."""
  torch.cuda.empty_cache()
  total = torch.cuda.get_device_properties(0).total_memory
  most = torch.cuda.memory_reserved() + (1 << 30)
  torch.cuda.set_per_process_memory_fraction(most / total)
  yield
  torch.cuda.set_per_process_memory_fraction(1.0)


def test_out_of_memory_is_torchs(small_memory):
  # Tensors that are a row or a value in memory: only what a call allocates is
  # large (8 GiB and more).
  x = torch.randn((1, 1024), device="cuda").expand(1 << 24, -1)
  ids = torch.zeros((1, 2), dtype=torch.int64, device="cuda")
  order = dense.sort_by_expert(ids, 2)
  wide = torch.randn((1, 1), device="cuda").expand(1, (1 << 31) - (1 << 17))
  for call in (lambda: dense.layer_norm(x),
               lambda: dense.layer_norm(x, return_stats=True),
               lambda: dense.tokens_to_experts(wide, order)):
    with pytest.raises(torch.OutOfMemoryError):
      call()
  # Nothing is left behind: the next call works.
  y = dense.layer_norm(x[:5])
  assert torch.equal(y[0], y[4])
