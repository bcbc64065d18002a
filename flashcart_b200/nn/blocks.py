"""Training blocks: element embedding, gated feed-forward and irreps dropout as modules.

They hold the parameters of the layers they stand for under the same names, so a checkpoint of
one loads into the other; :func:`use_training_blocks` puts them into a potential.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from flashcart_b200 import ops
from flashcart_b200.nn.layers import EquivariantGatedLayer, ProductPathWeights, _NoSpecialParameters


class ScaledEmbedding(nn.Module):
    """``offset + scale * weight[index]`` (parameter ``weight``, as ``nn.Embedding``); the
    gradient is summed over sorted tokens, so equal batches give equal gradients."""

    def __init__(self, n_types: int, features: int, scale: float = 1.0, offset: float = 0.0,
                 weight: Optional[nn.Parameter] = None):
        super().__init__()
        if n_types <= 0 or features <= 0:
            raise ValueError(f"n_types and features must be positive. Provided: {n_types}, {features}.")
        if weight is not None and tuple(weight.shape) != (n_types, features):
            raise ValueError(f"weight must be ({n_types}, {features}), got {tuple(weight.shape)}.")
        self.n_types, self.features = n_types, features
        self.scale, self.offset = float(scale), float(offset)
        self.weight = nn.Parameter(torch.randn(n_types, features)) if weight is None else weight

    @classmethod
    def stands_for(cls, emb: nn.Module) -> bool:
        """Whether ``emb`` is a plain table: a padding index, a norm limit, frequency scaling and
        sparse gradients are not this module's."""
        return (type(emb) is nn.Embedding and emb.padding_idx is None and emb.max_norm is None
                and not emb.scale_grad_by_freq and not emb.sparse)

    @classmethod
    def from_embedding(cls, emb: nn.Embedding, scale: float = 1.0, offset: float = 0.0) -> "ScaledEmbedding":
        """The same table (shared, not copied)."""
        if not cls.stands_for(emb):
            raise ValueError(f"ScaledEmbedding stands for plain embeddings only (no padding_idx, max_norm, "
                             f"scale_grad_by_freq or sparse gradients). Provided: {emb}.")
        return cls(emb.num_embeddings, emb.embedding_dim, scale, offset, weight=emb.weight)

    def forward(self, index: torch.Tensor) -> torch.Tensor:
        return ops.embedding(self.weight, index, self.scale, self.offset)

    def extra_repr(self) -> str:
        return f"{self.n_types}, {self.features}, scale={self.scale}, offset={self.offset}"


class IrrepsDropout(_NoSpecialParameters, nn.Module):
    """Dropout of whole irreps: one decision per (row, rank, channel), shared by the rank's
    components, so the layer commutes with rotations; identity in evaluation.

    Without a seed every training call draws the mask's 128 bits from torch's generator of the
    device, as ``nn.Dropout`` does: ``torch.manual_seed`` decides (ranks seeded apart drop
    apart), a restored generator state resumes the masks, and activation checkpointing, which
    restores it too, recomputes the same ones. With a seed the layer has a stream of its own,
    the device buffer ``rng`` = (key, calls so far), which is not part of the state dict; such
    a layer cannot tell which call a recomputation stands for and refuses to be recomputed."""

    def __init__(self, p: float, l_max: int = 0, seed: Optional[int] = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must lie in [0, 1]. Provided: {p}.")
        self.p, self.l_max = float(p), int(l_max)
        own = lambda *v: None if seed is None else torch.tensor(v, dtype=torch.int64)
        self.register_buffer("rng", own(0 if seed is None else int(seed), 0), persistent=False)
        self.register_buffer("advance", own(0, 1), persistent=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x
        # the gradient regenerates the mask from these two numbers
        if self.rng is None:
            state = torch.empty(2, dtype=torch.int64, device=x.device).random_()
        else:
            if not torch.compiler.is_compiling() and torch._C._current_graph_task_id() != -1:
                raise RuntimeError("IrrepsDropout with a seed of its own was called inside a backward (activation "
                                   "checkpointing?), where it would draw another mask than the forward did; leave "
                                   "the seed out to use torch's generator")
            state = self.rng.clone()
            self.rng.add_(self.advance)
        return ops.irreps_dropout(x, state, self.p, self.l_max)

    def extra_repr(self) -> str:
        return f"p={self.p}, l_max={self.l_max}"


class GatedFeedForward(EquivariantGatedLayer):
    """``EquivariantGatedLayer`` (reference ``nn/layers.py:543-648``: same constructor,
    parameters and result) whose gate map, value map, activation and product are one kernel,
    with one fused backward for all gradients; optionally dropout of the hidden irreps."""

    def __init__(self, l_max: int, in_features: int, hidden_features: Optional[int] = None,
                 gate_activation: str = "silu", gate_bias: bool = True, use_triton: bool = False,
                 dropout: float = 0.0, seed: Optional[int] = None):
        super().__init__(l_max, in_features, hidden_features, gate_activation, gate_bias, use_triton)
        self.dropout = IrrepsDropout(dropout, l_max, seed)
        self.register_buffer("scales", torch.cat([self.value_linear.scale.reshape(-1),
                                                  self.gate_linear.scale.reshape(1),
                                                  self.gate_activation.scale.reshape(1)]), persistent=False)

    @classmethod
    def from_layer(cls, layer: EquivariantGatedLayer, dropout: float = 0.0,
                   seed: Optional[int] = None) -> "GatedFeedForward":
        """The same parameters (shared, not copied)."""
        with torch.random.fork_rng(devices=[]):  # the initial weights drawn here are thrown away
            new = cls(layer.l_max, layer.in_features, layer.hidden_features, layer.gate_activation_name,
                      layer.gate_bias, dropout=dropout, seed=seed)
        new.value_linear, new.gate_linear = layer.value_linear, layer.gate_linear
        new.output_linear, new.gate_activation = layer.output_linear, layer.gate_activation
        new.scales = torch.cat([layer.value_linear.scale.reshape(-1), layer.gate_linear.scale.reshape(1),
                                layer.gate_activation.scale.reshape(1)])
        new.dropout.to(new.scales.device)
        new.train(layer.training)
        return new

    def forward(self, node_feats: torch.Tensor) -> torch.Tensor:
        if node_feats.shape[-1] != self.in_dim:
            raise RuntimeError(f"Incorrect last dimension for node_feats. Expected {self.in_dim}, "
                               f"got {node_feats.shape[-1]}.")
        dtype = node_feats.dtype
        cast = lambda w: w if w is None or w.dtype == dtype else w.to(dtype)
        acc = torch.float64 if dtype == torch.float64 else torch.float32
        hidden = ops.gated_feed_forward(node_feats, [cast(w) for w in self.value_linear.weight],
                                        cast(self.gate_linear.weight), cast(self.gate_linear.bias),
                                        self.scales.to(acc), self.l_max, self.gate_activation_name)
        return self.output_linear(self.dropout(hidden), residual=node_feats)


class _FusedPathWeights(ProductPathWeights):
    """Element-dependent path weights ``1 + delta[type]`` in one lookup."""

    def forward(self, atom_types=None):
        if atom_types is None:
            raise ValueError("atom_types required when n_elements is set.")
        return ops.embedding(self.delta.weight, atom_types, 1.0, 1.0)


def _layer_seed(seed: Optional[int], layer: int) -> Optional[int]:
    """A key of its own for every layer of every seed: the seeds' first keys lie far apart (seed
    times an odd number near 2^64 / 1.618, modulo 2^64), as signed 64-bit integers."""
    if seed is None:
        return None
    key = (int(seed) * 0x9E3779B97F4A7C15 + layer) % 2 ** 64
    return key - 2 ** 64 if key >= 2 ** 63 else key


def use_training_blocks(model: nn.Module, dropout: float = 0.0, seed: Optional[int] = None) -> nn.Module:
    """Put the training blocks into a :class:`~flashcart_b200.model.flashcart.FlashCartPotential`
    (in place; returned for convenience): the element embeddings, the element-dependent path
    weights and the gated layers. Parameters, their names and the model's results stay the
    same, up to rounding (embeddings with options that :class:`ScaledEmbedding` does not have stay
    as they are); ``dropout`` > 0 drops hidden irreps of the gated layers in training
    mode, from torch's generator or, with a ``seed``, from a stream of each layer (see
    :class:`IrrepsDropout`; give every rank of a data-parallel run a seed of its own)."""
    if ScaledEmbedding.stands_for(model.embedding):
        model.embedding = ScaledEmbedding.from_embedding(model.embedding)
    for inter in model.interactions:
        for name in ("emb_i", "emb_j"):
            if ScaledEmbedding.stands_for(getattr(inter, name)):
                setattr(inter, name, ScaledEmbedding.from_embedding(getattr(inter, name)))
    for product in model.products:
        for weights in product.path_weights:
            if weights.element_dependent and ScaledEmbedding.stands_for(weights.delta):
                weights.__class__ = _FusedPathWeights  # same attributes, another lookup
    if model.nonlinearity:
        for k, layer in enumerate(model.nonlinearities):
            model.nonlinearities[k] = GatedFeedForward.from_layer(layer, dropout, _layer_seed(seed, k))
    return model
