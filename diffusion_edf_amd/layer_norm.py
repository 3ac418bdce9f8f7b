"""EquivariantLayerNormV2 (reference ``equiformer/layer_norm.py:91-156``) with gradients, alone and fused with what stands between two blocks
(``gnn_block.py:164-218``): dropout of the block's output, its gate, the residual scale and the sum.  One kernel launch forward, and backward one plus the sums
of the parameters' gradients; HIP kernels ``dedf_norm_gate_residual(_backward)``."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from .drop import RowShape, TYPES, check_dropout, check_gpu, check_rows, launch, ptr, row_shape


def _struct(shape: RowShape, x, y, gate, scale, eps, post_w, post_b, next_w, next_b, p, rng) -> _lib.DedfNorm:
    return _lib.DedfNorm(TYPES[x.dtype], x.shape[0], len(shape.blocks), 1 if gate is None else gate.shape[0], shape.mul, shape.degree, x.data_ptr(), ptr(y), ptr(gate),
                         int(gate is not None and gate.dtype == torch.float32), scale, eps, ptr(post_w), ptr(post_b), ptr(next_w), ptr(next_b), p, ptr(rng))


def _forward(shape, x, y, gate, scale, eps, post_w, post_b, next_w, next_b, p, rng, keep_rng):
    a = _struct(shape, x, y, gate, scale, eps, post_w, post_b, next_w, next_b, p, rng)
    h = torch.empty_like(x) if y is not None else None
    z = torch.empty_like(x) if next_w is not None else None
    used = torch.empty(2, dtype=torch.int64, device=x.device) if keep_rng and p > 0.0 else None
    launch("dedf_norm_gate_residual", x.device, _lib.load().dedf_norm_gate_residual, C.byref(a), ptr(h), ptr(z), ptr(used))
    return h, z, used


class _NormGateResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, post_w, post_b, next_w, next_b, shape, scale, eps, p, rng):
        h, z, used = _forward(shape, x, y, gate, scale, eps, post_w, post_b, next_w, next_b, p, rng, True)
        ctx.save_for_backward(x, y, gate, post_w, post_b, next_w, next_b, used)
        ctx.rest = shape, scale, eps, p
        ctx.set_materialize_grads(False)
        return h, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_h, grad_z):
        x, y, gate, post_w, post_b, next_w, next_b, used = ctx.saved_tensors
        shape, scale, eps, p = ctx.rest
        if grad_h is None and grad_z is None:
            return (None,) * 12
        need = ctx.needs_input_grad
        grad_h, grad_z = (None if g is None else g.contiguous() for g in (grad_h, grad_z))
        a = _struct(shape, x, y, gate, scale, eps, post_w, post_b, next_w, next_b, p, used)
        d_x, d_y, d_gate = (torch.empty_like(t) if n else None for n, t in zip(need[:3], (x, y, gate)))
        params = [torch.empty_like(t) if n else None for n, t in zip(need[3:7], (post_w, post_b, next_w, next_b))]
        lib = _lib.load()
        scratch = torch.empty(lib.dedf_norm_scratch_bytes(C.byref(a)), dtype=torch.uint8, device=x.device)
        launch("dedf_norm_gate_residual_backward", x.device, lib.dedf_norm_gate_residual_backward, C.byref(a), ptr(grad_h), ptr(grad_z), ptr(d_x), ptr(d_y),
               ptr(d_gate), *map(ptr, params), scratch.data_ptr(), scratch.numel())
        return (d_x, d_y, d_gate, *params, None, None, None, None, None)


def _check_affine(name: str, weight, bias, shape: RowShape):
    if weight is None:
        if bias is not None:
            raise ValueError(f"{name}_bias without {name}_weight")
        return None, None
    if weight.dtype != torch.float32 or weight.shape != (shape.channels,):
        raise ValueError(f"{name}_weight: float32 ({shape.channels},), got {weight.dtype} {tuple(weight.shape)}")
    if bias is None or not shape.scalars:
        if shape.scalars:
            raise ValueError(f"{name}_bias: float32 ({shape.scalars},) for the channels of degree 0")
        if bias is not None and bias.numel():
            raise ValueError(f"{name}_bias: no channels of degree 0")
        return weight.contiguous(), None
    if bias.dtype != torch.float32 or bias.shape != (shape.scalars,):
        raise ValueError(f"{name}_bias: float32 ({shape.scalars},), got {bias.dtype} {tuple(bias.shape)}")
    return weight.contiguous(), bias.contiguous()


def _run(shape, x, y, gate, post_w, post_b, next_w, next_b, scale, eps, p, rng):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, gate, post_w, post_b, next_w, next_b)):
        return _NormGateResidual.apply(x, y, gate, post_w, post_b, next_w, next_b, shape, scale, eps, p, rng)
    return _forward(shape, x, y, gate, scale, eps, post_w, post_b, next_w, next_b, p, rng, False)[:2]


def norm_gate_residual(x: torch.Tensor, y: torch.Tensor, irreps, scale: float = 1.0, gate: Optional[torch.Tensor] = None,
                       post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None, dropout: float = 0.0,
                       rng: Optional[torch.Tensor] = None, next_weight: Optional[torch.Tensor] = None, next_bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """What stands between two blocks of a residual network on irreps features, ``x`` the stream and ``y`` the block's output, both ``(N, dim(irreps))``::

        u = LayerNorm(y; post_weight, post_bias)  (or y)       h = x + scale * gate * dropout(u)       z = LayerNorm(h; next_weight, next_bias)  (or None)

    -> ``(h, z)``.  ``gate`` ``(G, channels)`` multiplies all components of a channel; its rows belong to G runs of N / G consecutive rows: one row for a
    learned scale, one a pose, or one a node.  It has the features' type or float32; the norms' weights and biases are float32, biases for the channels of
    degree 0 only.  ``dropout`` drops whole channels, as ``equivariant_dropout`` with the same ``rng`` would.  Differentiable once."""
    shape = row_shape(irreps)
    check_rows("x", x, shape.width)
    if y.shape != x.shape or y.dtype != x.dtype:
        raise ValueError(f"y: {x.dtype} {tuple(x.shape)} like x, got {y.dtype} {tuple(y.shape)}")
    if gate is not None:
        if gate.ndim != 2 or gate.shape[1] != shape.channels or len(gate) == 0 or len(x) % len(gate):
            raise ValueError(f"gate: (G, {shape.channels}) with G a divisor of {len(x)} rows, got {tuple(gate.shape)}")
        if gate.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"gate: {x.dtype} or float32, got {gate.dtype}")
        if len(x) == 0:
            raise ValueError("gate: no rows")
        gate = gate.contiguous()
    post_weight, post_bias = _check_affine("post", post_weight, post_bias, shape)
    next_weight, next_bias = _check_affine("next", next_weight, next_bias, shape)
    if not eps >= 1e-30:
        raise ValueError(f"eps {eps}: at least 1e-30")
    p = check_dropout(dropout, rng, x.device)
    rng = rng.contiguous() if p > 0.0 else None
    check_gpu("norm_gate_residual", x, y, gate, post_weight, post_bias, next_weight, next_bias)
    return _run(shape, x.contiguous(), y.contiguous(), gate, post_weight, post_bias, next_weight, next_bias, float(scale), float(eps), p, rng)


def equivariant_layer_norm(x: torch.Tensor, irreps, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``EquivariantLayerNormV2.forward`` with affine parameters: the scalars centred over their channels, every degree divided by the root of its mean square."""
    shape = row_shape(irreps)
    check_rows("x", x, shape.width)
    weight, bias = _check_affine("next", weight, bias, shape)
    if weight is None:
        raise ValueError(f"weight: float32 ({shape.channels},)")
    if not eps >= 1e-30:
        raise ValueError(f"eps {eps}: at least 1e-30")
    check_gpu("equivariant_layer_norm", x, weight, bias)
    return _run(shape, x.contiguous(), None, None, None, None, weight, bias, 1.0, float(eps), 0.0, None)[1]


class EquivariantLayerNormV2(torch.nn.Module):
    """reference ``equiformer/layer_norm.py:64-156``: parameters ``affine_weight`` (one a channel) and ``affine_bias`` (degree 0)"""

    def __init__(self, irreps, eps: float = 1e-5):
        super().__init__()
        shape = row_shape(irreps)
        self.irreps, self.eps = irreps, eps
        self.affine_weight = torch.nn.Parameter(torch.ones(shape.channels))
        self.affine_bias = torch.nn.Parameter(torch.zeros(shape.scalars))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return equivariant_layer_norm(x, self.irreps, self.affine_weight, self.affine_bias if len(self.affine_bias) else None, self.eps)


class NormGateResidual(torch.nn.Module):
    """``norm_gate_residual`` with its parameters: ``post_norm`` and ``next_norm`` hold them under the names of ``EquivariantLayerNormV2``; either may be
    left out.  Dropout in training only; ``rng`` holds the seed and counts the training calls."""

    def __init__(self, irreps, scale: float = 1.0, post_norm: bool = True, next_norm: bool = True, drop_prob: float = 0.0, eps: float = 1e-5, seed: int = 0):
        super().__init__()
        self.irreps, self.scale, self.drop_prob, self.eps = irreps, scale, float(drop_prob), eps
        self.post_norm = EquivariantLayerNormV2(irreps, eps) if post_norm else None
        self.next_norm = EquivariantLayerNormV2(irreps, eps) if next_norm else None
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64), persistent=False)

    def forward(self, x: torch.Tensor, y: torch.Tensor, gate: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        p = self.drop_prob if self.training else 0.0
        affine = [None if n is None else t for n in (self.post_norm, self.next_norm) for t in ((None, None) if n is None else (n.affine_weight, n.affine_bias))]
        out = norm_gate_residual(x, y, self.irreps, self.scale, gate, affine[0], affine[1], p, self.rng, affine[2], affine[3], self.eps)
        if p > 0.0:
            self.rng[1] += 1
        return out
