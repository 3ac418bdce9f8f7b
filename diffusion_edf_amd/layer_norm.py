"""EquivariantLayerNormV2 (reference ``equiformer/layer_norm.py:91-156``) with gradients, alone and fused with what stands between two blocks
(``gnn_block.py:164-218``): dropout of the block's output, its gate, the residual scale and the sum.  One kernel launch forward, and backward one plus the sums
of the parameters' gradients; HIP kernels ``dedf_norm_gate_residual(_backward)``."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .drop import DrawsMasks, current_stream, row_shape


def norm_gate_residual(x: torch.Tensor, y: torch.Tensor, irreps, scale: float = 1.0, gate: Optional[torch.Tensor] = None,
                       post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None, dropout: float = 0.0,
                       rng: Optional[torch.Tensor] = None, next_weight: Optional[torch.Tensor] = None, next_bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """What stands between two blocks of a residual network on irreps features, ``x`` the stream and ``y`` the block's output, both ``(N, dim(irreps))``::

        u = LayerNorm(y; post_weight, post_bias)  (or y)       h = x + scale * gate * dropout(u)       z = LayerNorm(h; next_weight, next_bias)  (or None)

    -> ``(h, z)``.  ``gate`` ``(G, channels)`` multiplies all components of a channel; its rows belong to G runs of N / G consecutive rows: one row for a
    learned scale, one a pose, or one a node.  It has the features' type or float32; the norms' weights and biases are float32, biases for the channels of
    degree 0 only.  ``dropout`` drops whole channels, as ``equivariant_dropout`` with the same ``rng`` would.  Differentiable once."""
    h, z = _lib.ops().norm_gate_residual(x, y, row_shape(irreps).native, scale, gate, post_weight, post_bias, dropout, rng, next_weight, next_bias, eps, current_stream(x))
    return h, z


def equivariant_layer_norm(x: torch.Tensor, irreps, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``EquivariantLayerNormV2.forward`` with affine parameters: the scalars centred over their channels, every degree divided by the root of its mean square."""
    return _lib.ops().norm_gate_residual(x, None, row_shape(irreps).native, 1.0, None, None, None, 0.0, None, weight, bias, eps, current_stream(x))[1]


class EquivariantLayerNormV2(torch.nn.Module):
    """reference ``equiformer/layer_norm.py:64-156``: parameters ``affine_weight`` (one a channel) and ``affine_bias`` (degree 0)"""

    def __init__(self, irreps, eps: float = 1e-5):
        super().__init__()
        shape = row_shape(irreps)
        self.irreps, self.eps = irreps, eps
        self.affine_weight = torch.nn.Parameter(torch.ones(shape.channels))
        self.affine_bias = torch.nn.Parameter(torch.zeros(shape.scalars))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return equivariant_layer_norm(x, self.irreps, self.affine_weight.float(), self.affine_bias.float(), self.eps)          # (float32 after half() too)


class NormGateResidual(DrawsMasks):
    """``norm_gate_residual`` with its parameters: ``post_norm`` and ``next_norm`` hold them under the names of ``EquivariantLayerNormV2``; either may be
    left out.  Dropout in training only, masks as ``DrawsMasks`` has them."""

    def __init__(self, irreps, scale: float = 1.0, post_norm: bool = True, next_norm: bool = True, drop_prob: float = 0.0, eps: float = 1e-5, seed: Optional[int] = None):
        super().__init__()
        self.irreps, self.scale, self.drop_prob, self.eps = irreps, scale, float(drop_prob), eps
        self.post_norm = EquivariantLayerNormV2(irreps, eps) if post_norm else None
        self.next_norm = EquivariantLayerNormV2(irreps, eps) if next_norm else None
        self._start_masks(seed)

    def forward(self, x: torch.Tensor, y: torch.Tensor, gate: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        p = self.drop_prob if self.training else 0.0
        affine = [None if n is None else t for n in (self.post_norm, self.next_norm) for t in ((None, None) if n is None else (n.affine_weight.float(), n.affine_bias.float()))]
        out = norm_gate_residual(x, y, self.irreps, self.scale, gate, affine[0], affine[1], p, self._rng_at(x) if p > 0.0 else None, affine[2], affine[3], self.eps)
        if p > 0.0:
            self.rng[1] += 1
        return out
