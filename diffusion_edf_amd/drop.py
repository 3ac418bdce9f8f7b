"""Dropout in training: the random words that every operator of the package draws its masks from, and dropout of whole irreps channels.

No mask is ever stored.  An operator keeps an element where its Philox4x32-10 word -- key: the seed, counter: the element's place and the offset -- is at
least ``floor(p * 2**32)``, and its backward pass draws the same words again (``include/dedf.h`` lists the counters).  ``rng = [seed, offset]`` is an int64
tensor on the device: the kernels read it there, so a captured graph draws a new mask in each replay if the program changes the offset in between.  Two
calls with one ``rng`` draw the same words: give each call of a step a seed or an offset of its own.  The modules (``EquivariantDropout``, ``EdgeAttention``, ``NormGateResidual``) have a seed
each and count their calls (``DrawsMasks``); where a forward pass is run again for its activations, as in checkpointing, call the functions with an ``rng`` of your
own, which such a run repeats."""
from __future__ import annotations

import copy
import functools
from typing import List, Optional, Tuple

import torch

from . import _lib
from .so3 import parse_irreps

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
        self.native = _lib.ops().Shape([m for m, _ in self.blocks], [l for _, l in self.blocks], self.width, self.channels, self.scalars)


@functools.lru_cache(maxsize=256)
def _shape_of_text(irreps: str) -> RowShape:
    return RowShape(irreps)


def row_shape(irreps) -> RowShape:
    return _shape_of_text(irreps) if isinstance(irreps, str) else _shape_of_text("+".join(f"{m}x{l}e" for m, l in parse_irreps(irreps)))


def current_stream(x: torch.Tensor) -> int:
    """the current stream of the tensor's GPU, as the library takes it"""
    return torch._C._cuda_getCurrentRawStream(x.device.index) if x.is_cuda else 0


def equivariant_dropout(x: torch.Tensor, irreps, p: float, rng: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Drops whole channels (all ``2l+1`` components of one) of the rows ``(N, dim(irreps))`` with probability ``p`` and scales the others by ``1 / (1 - p)``
    (reference ``equiformer/drop.py:76-96`` in training mode).  float32, float16 or bfloat16; differentiable once."""
    return _lib.ops().equivariant_dropout(x, row_shape(irreps).native, p, rng, current_stream(x))


class DrawsMasks(torch.nn.Module):
    """What the modules with dropout have in common: ``rng = [seed, offset]`` on the module's device, the offset counting its training calls.  Without a seed
    every instance draws one from torch's generator, as its parameters' first values are drawn, so layers have masks of their own and ``torch.manual_seed`` repeats
    them; ``deepcopy`` draws again.  A seed that was given stays, in copies too.  ``rng`` is in no state dict (the reference's have no such entry): a program that resumes where it stopped
    saves and restores it beside them.  It is no buffer either: ``DistributedDataParallel`` would overwrite it on every rank with the first rank's; ranks that are to
    drop different places seed torch differently, or each give a seed."""

    def _start_masks(self, seed: Optional[int]) -> None:
        self.seed_drawn = seed is None
        self.rng = dropout_rng(_drawn_seed() if seed is None else seed, device="cpu")

    def _rng_at(self, x: torch.Tensor) -> torch.Tensor:
        if self.rng.device != x.device:
            self.rng = self.rng.to(x.device)
        return self.rng

    def _apply(self, fn, recurse: bool = True):
        super()._apply(fn, recurse)
        moved = fn(self.rng)
        if not (moved.is_meta or self.rng.is_meta):
            moved.copy_(self.rng)          # (to_empty() makes memory without values)
        self.rng = moved
        return self

    def __deepcopy__(self, memo):
        twin = self.__class__.__new__(self.__class__)
        memo[id(self)] = twin
        twin.__setstate__(copy.deepcopy(self.__dict__, memo))
        if twin.seed_drawn:
            twin.rng[0] = _drawn_seed()
        return twin


def _drawn_seed() -> int:
    return int(torch.empty((), dtype=torch.int64, device="cpu").random_())


class EquivariantDropout(DrawsMasks):
    """reference ``equiformer/drop.py:76-96``: identity in eval; masks as ``DrawsMasks`` has them"""

    def __init__(self, irreps, drop_prob: float, seed: Optional[int] = None):
        super().__init__()
        self.irreps, self.drop_prob = irreps, float(drop_prob)
        row_shape(irreps)
        self._start_masks(seed)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.training or self.drop_prob == 0.0:
            return x
        out = equivariant_dropout(x, self.irreps, self.drop_prob, self._rng_at(x))
        self.rng[1] += 1
        return out
