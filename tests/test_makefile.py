"""What the native build's targets need (no GPU, nothing is built)."""

import shutil
import subprocess

import pytest

from jax_tpu_embedding.sparsecore import _native


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
@pytest.mark.parametrize("targets,library,module", [
    ((), True, False), (("all",), True, False), (("python",), False, True),
    (("all", "python"), True, True)])
def test_targets(targets, library, module):
  """The library, for users of its C ABI, needs no Python and no torch."""
  out = subprocess.run(
      ["make", "-n", "-B", "-C", str(_native._PKG_ROOT / "csrc"), *targets],  # pylint: disable=protected-access
      check=True, capture_output=True, text=True).stdout
  assert ("libscemb.so" in out) == library
  assert ("torch" in out) == module and ("_dense.so" in out) == module
