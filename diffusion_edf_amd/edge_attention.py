"""The attention over a graph's edges in training: the last part of ``GraphAttentionMLP2.forward`` (reference ``graph_attention.py:237-273``) with gradients,
attention dropout and a learned bias for buckets of the edge length.  The edge lists are those of ``connectivity.py`` (sorted by destination); the
fused kernels of ``ScoreModelHead`` and ``UnetLayer`` evaluate the same attention for inference without per-edge tensors in memory.  HIP kernels:
``dedf_edge_attention(_backward)``."""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _lib
from .drop import DrawsMasks, current_stream


class EdgeSegments:
    """The edges' destinations ``edge_dst`` (int64, ascending, as ``radius_graph``, ``RadiusGraph`` and ``FpsPool`` return them) as the attention kernels
    read them: checked, in 32 bits, with the first edge of each of the ``n_dst`` rows.  Made once for a graph; waits for the check."""

    def __init__(self, edge_dst: torch.Tensor, n_dst: int):
        if edge_dst.ndim != 1 or edge_dst.dtype != torch.int64:
            raise ValueError(f"edge_dst: int64 (E,), got {edge_dst.dtype} {tuple(edge_dst.shape)}")
        n_dst = int(n_dst)
        if n_dst < 0 or (n_dst == 0 and len(edge_dst)):
            raise ValueError(f"{len(edge_dst)} edges to {n_dst} rows")
        if len(edge_dst) >= 1 << 31 or n_dst >= (1 << 31) - 1:
            raise NotImplementedError("fewer than 2**31 edges and rows")
        if not edge_dst.is_cuda:
            raise RuntimeError("EdgeSegments needs GPU tensors: the product has no CPU path")
        dev = edge_dst.device
        self.n_dst, self.n_edges, self.device = n_dst, len(edge_dst), dev
        self.dst = torch.empty(self.n_edges, dtype=torch.int32, device=dev)
        self.rowptr = torch.empty(n_dst + 1, dtype=torch.int32, device=dev)
        bad = torch.zeros(1, dtype=torch.int32, device=dev)
        edge_dst = edge_dst.contiguous()
        with torch.cuda.device(dev):
            rc = _lib.load().dedf_edge_segments(edge_dst.data_ptr(), self.n_edges, n_dst, self.dst.data_ptr(), self.rowptr.data_ptr(), bad.data_ptr(), current_stream(edge_dst))
        if rc != _lib.OK:
            raise RuntimeError(f"dedf_edge_segments failed ({rc})")
        if bad.item():
            raise ValueError(f"edge_dst is not ascending or leaves [0, {n_dst})")

    def __len__(self) -> int:
        return self.n_edges


def edge_attention(alpha: torch.Tensor, value: torch.Tensor, alpha_dot: torch.Tensor, segments: EdgeSegments, edge_logits: Optional[torch.Tensor] = None,
                   edge_length: Optional[torch.Tensor] = None, bias_boundaries: Optional[torch.Tensor] = None, bias_table: Optional[torch.Tensor] = None,
                   dropout: float = 0.0, rng: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention over the edges of each destination -> ``(n_dst, H, D)``::

        t[e, h] = sum_k SmoothLeakyReLU(alpha[e, h, k]) alpha_dot[h, k] + edge_logits[e] + bias_table[bucket(edge_length[e]), h]
        out[n, h] = sum over the edges e of n of softmax(t)[e, h] dropout value[e, h]

    ``alpha`` ``(E, H, K)`` and ``value`` ``(E, H, D)`` in float32, float16 or bfloat16 (views whose edges lie apart are read in place), ``alpha_dot``
    ``(H, K)`` or ``(1, H, K)``, ``edge_logits`` ``(E,)``, ``bias_table`` ``(B, H)`` with ``edge_length`` ``(E,)`` and ``B - 1`` ascending ``bias_boundaries``
    (bucket: the number of boundaries <= the length) in float32.  An edge and head whose logit is -inf takes no part, whatever ``alpha`` and ``value`` hold
    there; a row in which none does is zero.  The backward pass recomputes the probabilities from two numbers a row and head; gradients for ``alpha``, ``value``,
    ``alpha_dot``, ``edge_logits`` and ``bias_table``, once.  Results do not depend on the order in which anything ran."""
    return _lib.ops().edge_attention(alpha, value, alpha_dot, segments.dst, segments.rowptr, segments.n_dst, edge_logits, edge_length, bias_boundaries, bias_table, dropout, rng,
                                     current_stream(value))


class EdgeAttention(DrawsMasks):
    """``edge_attention`` with its parameters: ``alpha_dot`` ``(1, H, K)`` as in the reference's state dict (``graph_attention.py:139-214``) and, with
    ``bias_boundaries``, ``bias_table`` (zero at the start); after ``half()``, which rounds the parameters, they are used in float32 all the same, and the
    boundaries stay as they were, in float32: an edge keeps its bucket.  Dropout in training only, masks as ``DrawsMasks`` has them."""

    def __init__(self, num_heads: int, mul_alpha_head: int, alpha_drop: float = 0.0, bias_boundaries: Optional[Sequence[float]] = None, seed: Optional[int] = None):
        super().__init__()
        self.alpha_drop = float(alpha_drop)
        bound = math.sqrt(6.0 / (num_heads + mul_alpha_head))
        self.alpha_dot = torch.nn.Parameter(torch.empty(1, num_heads, mul_alpha_head).uniform_(-bound, bound))
        self.register_buffer("bias_boundaries", None if bias_boundaries is None else torch.as_tensor(bias_boundaries, dtype=torch.float32))
        self.bias_table = None if bias_boundaries is None else torch.nn.Parameter(torch.zeros(len(self.bias_boundaries) + 1, num_heads))
        self._start_masks(seed)

    def _apply(self, fn, recurse: bool = True):
        exact = self.bias_boundaries
        super()._apply(fn, recurse)
        if exact is not None and self.bias_boundaries.dtype != torch.float32:
            self.bias_boundaries = exact.to(self.bias_boundaries.device)
        return self

    def forward(self, alpha: torch.Tensor, value: torch.Tensor, segments: EdgeSegments, edge_logits: Optional[torch.Tensor] = None,
                edge_length: Optional[torch.Tensor] = None) -> torch.Tensor:
        p = self.alpha_drop if self.training else 0.0
        bias = {} if self.bias_table is None else {"edge_length": edge_length, "bias_boundaries": self.bias_boundaries, "bias_table": self.bias_table.float()}
        out = edge_attention(alpha, value, self.alpha_dot.float(), segments, edge_logits, dropout=p, rng=self._rng_at(value) if p > 0.0 else None, **bias)
        if p > 0.0:
            self.rng[1] += 1
        return out
