"""A ranking model with a mixture of experts, trained on synthetic clicks.

Tables and dense weights side by side: the lookup's activations of all
features go through layer norm to a router, every sample through its best
experts and back, and a last layer norm to a logit. The tables are updated by
embedding.tpu_sparse_dense_matmul_grad (Adagrad), everything else by
dense.adamw_update with moments of 8 or 32 bits; all gradients may be clipped to
a global norm before. Scoring can take the experts' weights in 8 bits.

  python -m jax_tpu_embedding.sparsecore.examples.ranking_moe --steps 100
"""

from __future__ import annotations

import argparse
import dataclasses
import math

import numpy as np

from jax_tpu_embedding.sparsecore import _native
from jax_tpu_embedding.sparsecore.lib.nn import dense
from jax_tpu_embedding.sparsecore.lib.nn import embedding
from jax_tpu_embedding.sparsecore.lib.nn import embedding_spec


@dataclasses.dataclass
class Config:
  batch: int = 1024
  features: int = 4
  vocabulary: int = 10_000
  dim: int = 16  # of a feature
  max_ids: int = 4  # of a feature and sample
  experts: int = 8
  choices: int = 2
  hidden: int = 64  # of an expert
  state_bits: int = 8
  learning_rate: float = 2e-3
  table_learning_rate: float = 0.05
  max_norm: float | None = None  # of all gradients
  seed: int = 0

  @property
  def width(self) -> int:
    return self.features * self.dim


class RankingModel:
  """Tables, dense weights and their optimizer states."""

  def __init__(self, config: Config):
    t = _native.require_gpu()
    c = self.config = config
    self.feature_specs = [
        embedding_spec.FeatureSpec(
            name=f"f{i}", input_shape=[c.batch, c.max_ids],
            output_shape=[c.batch, c.dim],
            table_spec=embedding_spec.TableSpec(
                name=f"t{i}", vocabulary_size=c.vocabulary,
                embedding_dim=c.dim, initializer=embedding_spec.normal(0.05),
                optimizer=embedding_spec.AdagradOptimizerSpec(
                    learning_rate=c.table_learning_rate), combiner="mean",
                max_ids_per_partition=c.batch * c.max_ids,
                max_unique_ids_per_partition=c.batch * c.max_ids))
        for i in range(c.features)]
    embedding.prepare_feature_specs_for_training(self.feature_specs, 1, 1)
    self.tables = embedding.init_embedding_variables(
        c.seed, embedding.get_table_specs(self.feature_specs),
        num_sparsecore_per_device=1)
    g = t.Generator(device="cuda").manual_seed(c.seed)
    new = lambda *shape: t.empty(shape, device="cuda").normal_(
        0.0, 1 / math.sqrt(shape[-2] if len(shape) > 1 else 1), generator=g)
    w = c.width
    self.weights = {
        "norm_in": t.ones(w, device="cuda"),
        "norm_in_bias": t.zeros(w, device="cuda"),
        "router": new(w, c.experts),
        "up": new(c.experts, w, c.hidden),
        "down": new(c.experts, c.hidden, w),
        "norm_out": t.ones(w, device="cuda"),
        "norm_out_bias": t.zeros(w, device="cuda"),
        "logit": new(w, 1),
    }
    for p in self.weights.values():
      p.requires_grad_()
    self.state = dense.init_adamw_state(
        list(self.weights.values()), state_bits=c.state_bits,
        decay=[p.dim() > 1 for p in self.weights.values()])

  def lookup(self, ids):
    """(preprocessed ids, a leaf of activations per feature)."""
    pre, _ = embedding.preprocess_sparse_dense_matmul_input(
        ids, None, self.feature_specs, 1, 1, num_sc_per_device=1)
    acts = embedding.tpu_sparse_dense_matmul(
        pre, self.tables, self.feature_specs, global_device_count=1,
        num_sc_per_device=1)
    return pre, [a.detach().requires_grad_() for a in acts]

  def logits(self, acts, experts_8=None):
    """A logit per sample from the features' activations. experts_8: the
    experts' weights in 8 bits (quantize_experts), for scoring."""
    t = _native.torch()
    c, w = self.config, self.weights
    x = dense.layer_norm(t.cat(acts, 1), w["norm_in"], w["norm_in_bias"])
    scores, ids = (x @ w["router"]).topk(c.choices, dim=1)
    # How many rows an expert gets stays on the GPU: nothing waits for it.
    order = dense.sort_by_expert(ids, c.experts)
    def product(rows, name):
      if experts_8 is None:
        return dense.expert_matmul(rows, w[name], order)
      return dense.matmul_8bit(rows, experts_8[name], order)
    rows = dense.tokens_to_experts(x, order)
    rows = product(t.relu(product(rows, "up")), "down")
    y = dense.tokens_from_experts(rows, scores.softmax(1), order)
    y = dense.layer_norm(x + y, w["norm_out"], w["norm_out_bias"])
    return (y @ w["logit"]).squeeze(1)

  def quantize_experts(self):
    """The experts' weights in 8 bits, once for many batches to score."""
    return {k: dense.quantize_weights(self.weights[k].detach())
            for k in ("up", "down")}

  def score(self, ids, experts_8=None):
    """The probability of a click per sample."""
    t = _native.torch()
    with t.no_grad():
      _, acts = self.lookup(ids)
      return self.logits(acts, experts_8).sigmoid()

  def step(self, ids, clicks):
    """One training step; returns the loss before it."""
    t = _native.torch()
    pre, acts = self.lookup(ids)
    loss = t.nn.functional.binary_cross_entropy_with_logits(
        self.logits(acts), clicks)
    params = list(self.weights.values())
    grads = t.autograd.grad(loss, acts + params)
    of_acts, of_params = list(grads[:len(acts)]), grads[len(acts):]
    factor = None
    if self.config.max_norm is not None:
      _, factor = dense.gradient_norm(grads, max_norm=self.config.max_norm)
      of_acts = [g * factor for g in of_acts]
    self.tables = embedding.tpu_sparse_dense_matmul_grad(
        of_acts, pre, self.tables, self.feature_specs, global_device_count=1,
        num_sc_per_device=1)
    dense.adamw_update(params, of_params, self.state,
                       learning_rate=self.config.learning_rate,
                       grad_scale=factor)
    return loss.detach()


class Clicks:
  """Batches of ids and whether the sample was clicked: each id of each
  feature has a hidden weight, and their sum decides."""

  def __init__(self, config: Config):
    self.config = config
    self._rng = np.random.default_rng(config.seed)
    self._hidden = self._rng.normal(
        size=(config.features, config.vocabulary)).astype(np.float32)

  def batch(self):
    t = _native.torch()
    c = self.config
    ids = [(self._rng.zipf(1.3, size=(c.batch, c.max_ids)) %
            c.vocabulary).astype(np.int32) for _ in range(c.features)]
    score = sum(self._hidden[i][x].mean(1) for i, x in enumerate(ids))
    return ids, t.from_numpy((score > 0).astype(np.float32)).cuda()


def train(config: Config, steps: int) -> list[float]:
  """The loss before each step."""
  model, clicks = RankingModel(config), Clicks(config)
  losses = [model.step(*clicks.batch()) for _ in range(steps)]
  return [float(x) for x in losses]


def main():
  parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
  parser.add_argument("--steps", type=int, default=100)
  parser.add_argument("--batch", type=int, default=Config.batch)
  parser.add_argument("--state_bits", type=int, default=Config.state_bits,
                      choices=(8, 32))
  parser.add_argument("--max_norm", type=float, default=None)
  args = parser.parse_args()
  losses = train(Config(batch=args.batch, state_bits=args.state_bits,
                        max_norm=args.max_norm), args.steps)
  for i in range(0, len(losses), max(1, len(losses) // 10)):
    print(f"step {i}: loss {losses[i]:.4f}")
  print(f"step {len(losses) - 1}: loss {losses[-1]:.4f}")


if __name__ == "__main__":
  main()
