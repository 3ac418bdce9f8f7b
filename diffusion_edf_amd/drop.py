"""Dropout in training: the random words that every operator of the package draws its masks from, and dropout of whole irreps channels.

No mask is ever stored.  An operator keeps an element where its Philox4x32-10 word -- key: the seed, counter: the element's place and the offset -- is at
least ``floor(p * 2**32)``, and its backward pass draws the same words again (``include/dedf.h`` lists the counters).  ``rng = [seed, offset]`` is an int64
tensor on the device: the kernels read it there, so a captured graph draws a new mask in each replay if the program changes the offset in between.  Two
calls with one ``rng`` draw the same words: give each call of a step an offset of its own (``EquivariantDropout`` and ``EdgeAttention`` count theirs)."""
from __future__ import annotations

import ctypes as C
import functools
from typing import List, Optional, Tuple

import torch

from . import _lib
from .so3 import parse_irreps

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}          # DEDF_F32, DEDF_F16, DEDF_BF16


def dropout_rng(seed: int, offset: int = 0, device="cuda") -> torch.Tensor:
    """``[seed, offset]`` on the device, what the ``rng`` argument of the operators takes"""
    return torch.tensor([seed, offset], dtype=torch.int64, device=device)


class RowShape:
    """irreps of a feature row as the row kernels take them: up to 4 blocks of ascending degree"""

    def __init__(self, irreps):
        self.blocks: List[Tuple[int, int]] = [(m, l) for m, l in parse_irreps(irreps) if m != 0]
        if not self.blocks or any(m < 0 for m, _ in self.blocks) or any(b[1] <= a[1] for a, b in zip(self.blocks, self.blocks[1:])):
            raise ValueError(f"irreps {irreps}: blocks of ascending degree")
        self.width = sum(m * (2 * l + 1) for m, l in self.blocks)
        self.channels = sum(m for m, _ in self.blocks)
        self.scalars = self.blocks[0][0] if self.blocks[0][1] == 0 else 0
        if len(self.blocks) > 4 or self.width > 2048 or self.blocks[-1][1] > 7:
            raise NotImplementedError(f"irreps {irreps}: at most 4 degrees up to 7 and 2048 components")
        pad = [(0, 0)] * (4 - len(self.blocks))
        self.mul = (C.c_int * 4)(*[m for m, _ in self.blocks + pad])
        self.degree = (C.c_int * 4)(*[l for _, l in self.blocks + pad])


@functools.lru_cache(maxsize=256)
def _shape_of_text(irreps: str) -> RowShape:
    return RowShape(irreps)


def row_shape(irreps) -> RowShape:
    return _shape_of_text(irreps) if isinstance(irreps, str) else _shape_of_text("+".join(f"{m}x{l}e" for m, l in parse_irreps(irreps)))


def check_rows(name: str, x: torch.Tensor, width: int) -> None:
    if x.ndim != 2 or x.shape[1] != width:
        raise ValueError(f"{name}: expected (rows, {width}), got {tuple(x.shape)}")
    if x.dtype not in TYPES:
        raise TypeError(f"{name}: float32, float16 or bfloat16, got {x.dtype}")
    if len(x) >= 1 << 31:
        raise NotImplementedError(f"{name}: fewer than 2**31 rows")


def check_dropout(p: float, rng: Optional[torch.Tensor], device: torch.device) -> float:
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout probability {p}: in [0, 1)")
    if p > 0.0:
        if rng is None:
            raise ValueError("dropout needs rng, an int64 tensor [seed, offset] (dropout_rng)")
        if rng.dtype != torch.int64 or rng.shape != (2,):
            raise ValueError(f"rng: int64 [seed, offset], got {rng.dtype} {tuple(rng.shape)}")
        if rng.device != device:
            raise ValueError(f"rng on {rng.device}, the features on {device}")
    return p


def check_gpu(what: str, *tensors) -> torch.device:
    """-> the one GPU that all tensors (None among them) are on"""
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on different devices")
    if dev.type != "cuda":
        raise RuntimeError(f"{what} needs GPU tensors: the product has no CPU path")
    return dev


def launch(what: str, device: torch.device, call, *args) -> None:
    """``call(*args, stream)`` on the device's current stream (with the device current: the library launches there); raises for what it returns"""
    if device.index == torch.cuda.current_device():
        rc = call(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            rc = call(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc != _lib.OK:
        raise (ValueError if rc == _lib.ERR_INVALID else NotImplementedError if rc == _lib.ERR_UNSUPPORTED else RuntimeError)(f"{what} failed ({rc})")


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _launch(x: torch.Tensor, shape: RowShape, p: float, rng: Optional[torch.Tensor], keep_rng: bool):
    out = torch.empty_like(x)
    used = torch.empty(2, dtype=torch.int64, device=x.device) if keep_rng else None
    launch("dedf_channel_dropout", x.device, _lib.load().dedf_channel_dropout, TYPES[x.dtype], x.shape[0], len(shape.blocks), shape.mul, shape.degree,
           x.data_ptr(), p, ptr(rng), out.data_ptr(), ptr(used))
    return out, used


class _EquivariantDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, shape, p, rng):
        out, used = _launch(x, shape, p, rng, True)
        ctx.save_for_backward(used)
        ctx.shape, ctx.p = shape, p
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _launch(grad.contiguous(), ctx.shape, ctx.p, ctx.saved_tensors[0], False)[0], None, None, None


def equivariant_dropout(x: torch.Tensor, irreps, p: float, rng: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Drops whole channels (all ``2l+1`` components of one) of the rows ``(N, dim(irreps))`` with probability ``p`` and scales the others by ``1 / (1 - p)``
    (reference ``equiformer/drop.py:76-96`` in training mode).  float32, float16 or bfloat16; differentiable once."""
    shape = row_shape(irreps)
    check_rows("x", x, shape.width)
    p = check_dropout(p, rng, x.device)
    check_gpu("equivariant_dropout", x, rng)
    if p == 0.0:
        return x
    x, rng = x.contiguous(), rng.contiguous()
    if torch.is_grad_enabled() and x.requires_grad:
        return _EquivariantDropout.apply(x, shape, p, rng)
    return _launch(x, shape, p, rng, False)[0]


class EquivariantDropout(torch.nn.Module):
    """reference ``equiformer/drop.py:76-96``: identity in eval.  ``rng`` (a buffer that is not saved) holds the seed and counts the training calls."""

    def __init__(self, irreps, drop_prob: float, seed: int = 0):
        super().__init__()
        self.irreps, self.drop_prob = irreps, float(drop_prob)
        row_shape(irreps)
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64), persistent=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.training or self.drop_prob == 0.0:
            return x
        out = equivariant_dropout(x, self.irreps, self.drop_prob, self.rng)
        self.rng[1] += 1
        return out
