"""The attention over a graph's edges in training: the last part of ``GraphAttentionMLP2.forward`` (reference ``graph_attention.py:237-273``) with gradients,
attention dropout and a learned bias for buckets of the edge length.  The edge lists are those of ``connectivity.py`` (sorted by destination); the
fused kernels of ``ScoreModelHead`` and ``UnetLayer`` evaluate the same attention for inference without per-edge tensors in memory.  HIP kernels:
``dedf_edge_attention(_backward)``."""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import torch

from . import _lib
from .drop import TYPES, check_dropout, check_gpu, launch, ptr


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
        dev = check_gpu("EdgeSegments", edge_dst)
        self.n_dst, self.n_edges, self.device = n_dst, len(edge_dst), dev
        self.dst = torch.empty(self.n_edges, dtype=torch.int32, device=dev)
        self.rowptr = torch.empty(n_dst + 1, dtype=torch.int32, device=dev)
        bad = torch.zeros(1, dtype=torch.int32, device=dev)
        edge_dst = edge_dst.contiguous()
        launch("dedf_edge_segments", dev, _lib.load().dedf_edge_segments, ptr(edge_dst), self.n_edges, n_dst, ptr(self.dst), ptr(self.rowptr), ptr(bad))
        if bad.item():
            raise ValueError(f"edge_dst is not ascending or leaves [0, {n_dst})")

    def __len__(self) -> int:
        return self.n_edges


def _rows(x: torch.Tensor) -> torch.Tensor:
    """the tensor itself where an edge's (heads, channels) lie together, whatever the distance of two edges, else a copy"""
    E, H, K = x.shape
    inner = (K == 1 or x.stride(2) == 1) and (H == 1 or x.stride(1) == K)
    return x if inner and x.stride(0) >= 0 else x.contiguous()


def _struct(seg: EdgeSegments, alpha, value, alpha_dot, logits, length, bounds, table, p, rng) -> _lib.DedfEdgeAttn:
    return _lib.DedfEdgeAttn(seg.n_edges, seg.n_dst, alpha.shape[1], alpha.shape[2], value.shape[2], TYPES[value.dtype], 0 if table is None else table.shape[0],
                             ptr(alpha), alpha.stride(0), ptr(value), value.stride(0), ptr(alpha_dot), ptr(seg.dst), ptr(seg.rowptr), ptr(logits), ptr(length),
                             ptr(bounds), ptr(table), p, ptr(rng))


def _forward(seg, alpha, value, alpha_dot, logits, length, bounds, table, p, rng, train):
    a = _struct(seg, alpha, value, alpha_dot, logits, length, bounds, table, p, rng)
    lib, dev = _lib.load(), value.device
    H, D = value.shape[1:]
    out = torch.empty(seg.n_dst, H, D, dtype=value.dtype, device=dev)
    out_f = norm = used = None
    if train:
        out_f = torch.empty(seg.n_dst, H, D, dtype=torch.float32, device=dev) if value.dtype != torch.float32 else None
        norm = torch.empty(seg.n_dst, H, 2, dtype=torch.float64, device=dev)
        used = torch.empty(2, dtype=torch.int64, device=dev) if p > 0.0 else None
    scratch = torch.empty(lib.dedf_edge_attention_scratch_bytes(C.byref(a), 0), dtype=torch.uint8, device=dev)
    launch("dedf_edge_attention", dev, lib.dedf_edge_attention, C.byref(a), ptr(out), ptr(out_f), ptr(norm), ptr(used), ptr(scratch), scratch.numel())
    return out, out_f, norm, used


class _EdgeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, alpha, value, alpha_dot, logits, table, seg, length, bounds, p, rng):
        out, out_f, norm, used = _forward(seg, alpha, value, alpha_dot, logits, length, bounds, table, p, rng, True)
        ctx.save_for_backward(alpha, value, alpha_dot, logits, table, length, bounds, out if out_f is None else out_f, norm, used)
        ctx.seg, ctx.p = seg, p
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        alpha, value, alpha_dot, logits, table, length, bounds, out_f, norm, used = ctx.saved_tensors
        seg, need, dev = ctx.seg, ctx.needs_input_grad, value.device
        a = _struct(seg, alpha, value, alpha_dot, logits, length, bounds, table, ctx.p, used)
        grad = grad.contiguous()
        d_alpha = torch.empty(alpha.shape, dtype=alpha.dtype, device=dev) if need[0] else None
        d_value = torch.empty(value.shape, dtype=value.dtype, device=dev) if need[1] else None
        d_dot, d_logits, d_table = (torch.empty_like(t) if n else None for n, t in zip(need[2:5], (alpha_dot, logits, table)))
        lib = _lib.load()
        scratch = torch.empty(lib.dedf_edge_attention_scratch_bytes(C.byref(a), 1), dtype=torch.uint8, device=dev)
        launch("dedf_edge_attention_backward", dev, lib.dedf_edge_attention_backward, C.byref(a), ptr(norm), ptr(out_f), ptr(grad), ptr(d_alpha), ptr(d_value),
               ptr(d_dot), ptr(d_logits), ptr(d_table), ptr(scratch), scratch.numel())
        return d_alpha, d_value, d_dot, d_logits, d_table, None, None, None, None, None


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
    if alpha.ndim != 3 or value.ndim != 3 or alpha.shape[:2] != value.shape[:2]:
        raise ValueError(f"alpha (E, H, K) and value (E, H, D): got {tuple(alpha.shape)} and {tuple(value.shape)}")
    if value.dtype not in TYPES or alpha.dtype != value.dtype:
        raise TypeError(f"alpha and value: both float32, float16 or bfloat16, got {alpha.dtype} and {value.dtype}")
    E, H, K = alpha.shape
    if min(H, K, value.shape[2]) < 1:
        raise ValueError(f"alpha {tuple(alpha.shape)}, value {tuple(value.shape)}: empty rows")
    if E != segments.n_edges:
        raise ValueError(f"{E} edges, the segments hold {segments.n_edges}")
    if alpha_dot.ndim == 3 and alpha_dot.shape[0] == 1:
        alpha_dot = alpha_dot[0]
    if alpha_dot.shape != (H, K) or alpha_dot.dtype != torch.float32:
        raise ValueError(f"alpha_dot: float32 ({H}, {K}), got {alpha_dot.dtype} {tuple(alpha_dot.shape)}")
    if edge_logits is not None and (edge_logits.shape != (E,) or edge_logits.dtype != torch.float32):
        raise ValueError(f"edge_logits: float32 ({E},), got {edge_logits.dtype} {tuple(edge_logits.shape)}")
    if bias_table is None:
        if edge_length is not None or bias_boundaries is not None:
            raise ValueError("edge_length and bias_boundaries come with bias_table")
    else:
        if bias_table.ndim != 2 or bias_table.shape[1] != H or len(bias_table) < 1 or bias_table.dtype != torch.float32:
            raise ValueError(f"bias_table: float32 (B, {H}), got {bias_table.dtype} {tuple(bias_table.shape)}")
        if edge_length is None or edge_length.shape != (E,) or edge_length.dtype != torch.float32:
            raise ValueError(f"edge_length: float32 ({E},)")
        if len(bias_table) > 1 and (bias_boundaries is None or bias_boundaries.shape != (len(bias_table) - 1,) or bias_boundaries.dtype != torch.float32):
            raise ValueError(f"bias_boundaries: float32 ({len(bias_table) - 1},)")
        if len(bias_table) == 1:
            bias_boundaries = None
    if H > 16 or H * K > 256 or H * value.shape[2] > 1024 or (bias_table is not None and (len(bias_table) > 1024 or bias_table.numel() > 2048)):
        raise NotImplementedError("at most 16 heads, 256 attention features and 1024 value channels an edge, 1024 buckets, 2048 bias entries")
    p = check_dropout(dropout, rng, value.device)
    dev = check_gpu("edge_attention", value, alpha, alpha_dot, edge_logits, edge_length, bias_boundaries, bias_table)
    if segments.device != dev:
        raise ValueError(f"segments on {segments.device}, the features on {dev}")
    alpha, value = _rows(alpha), _rows(value)
    alpha_dot, edge_logits, edge_length, bias_boundaries, bias_table = (None if t is None else t.contiguous() for t in (alpha_dot, edge_logits, edge_length, bias_boundaries, bias_table))
    rng = rng.contiguous() if p > 0.0 else None
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (alpha, value, alpha_dot, edge_logits, bias_table)):
        return _EdgeAttention.apply(alpha, value, alpha_dot, edge_logits, bias_table, segments, edge_length, bias_boundaries, p, rng)
    return _forward(segments, alpha, value, alpha_dot, edge_logits, edge_length, bias_boundaries, bias_table, p, rng, False)[0]


class EdgeAttention(torch.nn.Module):
    """``edge_attention`` with its parameters: ``alpha_dot`` ``(1, H, K)`` as in the reference's state dict (``graph_attention.py:139-214``) and, with
    ``bias_boundaries``, ``bias_table`` (zero at the start).  Dropout in training only; ``rng`` holds the seed and counts the training calls."""

    def __init__(self, num_heads: int, mul_alpha_head: int, alpha_drop: float = 0.0, bias_boundaries: Optional[Sequence[float]] = None, seed: int = 0):
        super().__init__()
        self.alpha_drop = float(alpha_drop)
        bound = math.sqrt(6.0 / (num_heads + mul_alpha_head))
        self.alpha_dot = torch.nn.Parameter(torch.empty(1, num_heads, mul_alpha_head).uniform_(-bound, bound))
        self.register_buffer("bias_boundaries", None if bias_boundaries is None else torch.as_tensor(bias_boundaries, dtype=torch.float32))
        self.bias_table = None if bias_boundaries is None else torch.nn.Parameter(torch.zeros(len(self.bias_boundaries) + 1, num_heads))
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64), persistent=False)

    def forward(self, alpha: torch.Tensor, value: torch.Tensor, segments: EdgeSegments, edge_logits: Optional[torch.Tensor] = None,
                edge_length: Optional[torch.Tensor] = None) -> torch.Tensor:
        p = self.alpha_drop if self.training else 0.0
        bias = {} if self.bias_table is None else {"edge_length": edge_length, "bias_boundaries": self.bias_boundaries, "bias_table": self.bias_table}
        out = edge_attention(alpha, value, self.alpha_dot, segments, edge_logits, dropout=p, rng=self.rng, **bias)
        if p > 0.0:
            self.rng[1] += 1
        return out
