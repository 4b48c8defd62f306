"""Transformer layers on the token operators of :mod:`blades_amd.ops`.

Drop-in subclasses: same parameters, same state-dict keys.  ``fused_norm`` and
``act_bits`` of the transformer models choose between these and the torch
layers.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from blades_amd import ops


class FusedLayerNorm(nn.LayerNorm):
    """:func:`blades_amd.ops.layer_norm` over the last axis."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return ops.layer_norm(x, self.weight, self.bias, self.eps)


class Act8Linear(nn.Linear):
    """Linear layer that keeps its input in 8 bits for the backward pass."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return ops.linear_act8(x, self.weight, self.bias)


def layer_types(fused_norm: bool = False, act_bits: int = 32):
    """(norm class, linear class, gelu function) of an encoder layer.

    ``act_bits``: bits in which the encoder's linear layers and GELUs keep
    their inputs for the backward pass: 32 (as they are) or 8.
    """
    if act_bits not in (8, 32):
        raise ValueError(f"act_bits must be 8 or 32, got {act_bits}")
    norm = FusedLayerNorm if fused_norm else nn.LayerNorm
    if act_bits == 8:
        return norm, Act8Linear, ops.gelu_act8
    return norm, nn.Linear, F.gelu


def head_loss(features: torch.Tensor, head: nn.Linear,
              targets: torch.Tensor) -> torch.Tensor:
    """Mean cross entropy of ``head(features)`` without its logits."""
    return ops.linear_cross_entropy(features, head.weight, targets, head.bias)
