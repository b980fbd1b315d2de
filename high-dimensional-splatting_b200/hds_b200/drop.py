"""Dropout from a counter-based generator: the mask follows from (seed, offset) alone, is drawn anew by
the backward, and is never stored.  No counterpart in the reference."""
from __future__ import annotations

import warnings

import torch

from . import gaussian_rasterizer as _ext
from . import rasterizer


class Dropout(torch.autograd.Function):
    """y = dropout(x); the backward is the same kernel on dL/dy under the same draw."""

    @staticmethod
    def forward(ctx, x, how):
        """how: dropout()'s (p, seed, offset, rows, draw)."""
        ctx.how = how[:-1]
        ctx.save_for_backward(how[-1])
        return _ext.dropout(x, *how)

    @staticmethod
    def backward(ctx, grad):
        draw, = ctx.saved_tensors  # raises if it has changed since
        p, seed, offset, rows = ctx.how
        return dropout(grad, p, seed=seed, offset=offset, rows=rows, draw=draw), None


def draw_numbers(p: float, seed: int | None, offset: int | None, draw: torch.Tensor | None) -> tuple[int, int]:
    """(seed, offset), 0 for those not given; warns when a mask would depend on nothing that was given."""
    if seed is None and offset is None and draw is None and 0 < p < 1:
        warnings.warn("dropout without seed, offset or draw takes the mask of (0, 0): the same at every call and in "
                      "every layer", stacklevel=3)
    return seed or 0, offset or 0


def dropout(x: torch.Tensor, p: float, *, seed: int | None = None, offset: int | None = None, rows: bool = False,
            draw: torch.Tensor | None = None) -> torch.Tensor:
    """x (float32, bfloat16 or float16) with each element zeroed with probability p (a multiple of
    1/65536) and the others scaled by the reciprocal of the kept share.  rows: whole rows along the last
    dimension are dropped together -- whole gaussians of an [N, C] tensor.

    The mask follows from (seed, offset) alone, which are 0 when not given: give every step and every use
    numbers of its own (a step counter as the offset, say), or they all drop the same elements.  A call
    that gives neither, nor draw, warns.  draw: an int64 tensor [2] = (seed, offset) on the device, used instead
    of the two numbers and read when the kernel runs, so that a captured graph can advance it; it must not
    change between a forward and its backward.  A p that rounds to 0 returns x itself."""
    if _ext.drop_threshold(p) == 0:
        return x
    seed, offset = draw_numbers(p, seed, offset, draw)
    x = x.contiguous()
    if rasterizer.needs_node(x):
        return Dropout.apply(x, (p, seed, offset, rows, draw))
    return _ext.dropout(x, p, seed, offset, rows, draw)
