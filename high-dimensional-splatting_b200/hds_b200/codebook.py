"""Codebook features: the lookup of per-gaussian features in a table, and its gradient.

A compact model holds a codebook [V, C] and one codeword id per gaussian instead of an [N, C] feature
table.  ``embedding`` gives the [N, C] features that ``rasterize`` blends; its backward sums the blend's
feature gradient by codeword.  No counterpart in the reference, whose models hold a feature row per
gaussian.
"""
from __future__ import annotations

import torch

from . import gaussian_rasterizer as _ext
from . import rasterizer
from .drop import draw_numbers


class Embedding(torch.autograd.Function):
    """scale * table[ids] with optional dropout; the backward returns dL/dtable in the table's type.

    Under hds_b200.rasterizer.accumulate_leaf_grads() (active during this forward), when table is a leaf
    that already holds a contiguous float32 .grad of its shape, the backward adds into that buffer and
    hands autograd no gradient for it (hooks on the table do not see that gradient; forwards that share the
    table then belong on one stream)."""

    @staticmethod
    def forward(ctx, table, ids, dtype, how):
        """how: embedding()'s (scale, padding_id, dropout_p, seed, offset, draw)."""
        scale, padding_id, dropout_p, seed, offset, draw = how
        out = _ext.embedding(table, ids, dtype, *how)
        ctx.leaf = table if (rasterizer.ACCUMULATE_INTO_LEAF_GRAD and table.is_leaf) else None
        ctx.table = (table.shape, table.dtype)
        # The backward's numbers, checked above.
        threshold, seed, offset, _ = _ext._draw(dropout_p, seed, offset, draw, table.device)
        ctx.how = (scale, padding_id, threshold, seed, offset)
        ctx.save_for_backward(ids, draw if threshold else None)
        return out

    @staticmethod
    def backward(ctx, grad):
        if (grad.requires_grad and torch.is_grad_enabled()) or rasterizer.has_tangent(grad):
            raise RuntimeError("the gradient of embedding() cannot be differentiated again")
        ids, draw = ctx.saved_tensors  # raises if the ids or the draw have changed since
        shape, dtype = ctx.table
        grad = grad.contiguous()
        # What hooks on saved tensors or an assignment to .data have put in their place goes to a kernel as
        # an address.
        _ext._check_ids(ids, grad.device)
        if ids.shape != grad.shape[:-1]:
            raise RuntimeError(f"ids were {tuple(grad.shape[:-1])} in the forward, and are {tuple(ids.shape)} now")
        how = (*ctx.how, _ext._draw_address(draw, grad.device))
        target = ctx.leaf.grad if ctx.leaf is not None else None
        if (target is not None and grad.dtype == torch.float32 and target.dtype == torch.float32
                and target.is_contiguous() and target.shape == shape and target.device == grad.device):
            _ext._sum_by_id(grad, ids, target, 1, *how)
            return None, None, None, None
        grad_table = torch.empty(shape, dtype=dtype, device=grad.device)
        _ext._sum_by_id(grad, ids, grad_table, 0, *how)
        return grad_table, None, None, None


def embedding(table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0, padding_id: int | None = None,
              dtype: torch.dtype | None = None, dropout_p: float = 0.0, seed: int | None = None,
              offset: int | None = None, draw: torch.Tensor | None = None) -> torch.Tensor:
    """scale * table[ids]: the features [*ids.shape, C] of the codeword ids under the codebook table
    [V, C] (float32, bfloat16 or float16; ids int32 or int64), in `dtype` (the table's type, or float32:
    the type rasterize takes).  Differentiable in table; the same backward call gives the same bits.
    scale, times the reciprocal of the kept share, must be finite in float32.

    padding_id: ids with this value (a negative one, say, for gaussians without a codeword) give rows of
    zeros and no gradient.  Any other id outside [0, V) does too, and sets native.device_status().

    dropout_p: drops elements of the result with this probability (a multiple of 1/65536) and scales the
    others up, in the same pass.  The mask follows from (seed, offset) alone (0 when not given; a call that
    gives neither, nor draw, warns): give every step and use its own, a step counter, say, as the offset.
    It is drawn anew in the backward, never stored.  draw: an int64 tensor [2] = (seed, offset) on the
    device, used instead of the two numbers and read when the kernels run, so that a captured graph can
    advance it; it must not change between a forward and its backward.

    To capture a backward pass into a CUDA graph, keep no eager autograd graph of the same table alive
    (torch ties the leaf's gradient to the stream of the first one); gaussian_rasterizer.embedding_backward
    has no such rule."""
    seed, offset = draw_numbers(dropout_p, seed, offset, draw)
    table = table.contiguous()
    ids = ids.contiguous()
    if rasterizer.needs_node(table):
        return Embedding.apply(table, ids, dtype, (scale, padding_id, dropout_p, seed, offset, draw))
    return _ext.embedding(table, ids, dtype, scale, padding_id, dropout_p, seed, offset, draw)
