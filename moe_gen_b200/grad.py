"""Differentiable forms of the layer's steps around the experts, for what is trained while the experts stay as they are: a
router calibrated behind quantising them, adapters on the expert-sorted rows.  Each is a torch.autograd.Function over the
layer's own kernels, forward and backward.  The reference has no training path (DeepseekV3MoE.forward runs moe_infer only,
modeling_deepseek_v3.py:614-626).

    idx, w = route(layer, logits)                                # w is differentiable in logits
    counts, _, pad, dst = layer.permute_plan(idx)
    rows = sort_rows(layer, x, dst, layer.padded_rows(idx.numel()), counts, pad)
    ...                                                          # experts, adapters on rows
    y = combine_rows(layer, out_rows, dst, idx, w, counts, pad, shared_out)

A step can be captured into a CUDA graph, its backward pass too; as with any torch step, no eager graph of the same leaves may be alive
then (torch's accumulation nodes belong to the stream that they were made on).
"""
from typing import Optional, Tuple

import torch

from .layer import MoELayer, _whole


# Gradients are taken through _whole: torch hands them over as they come, and the backward of cat and of flat views cuts them out of a
# larger tensor at any element.
class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, layer):
        idx, w = layer.route_topk(logits)
        ctx.layer = layer
        ctx.save_for_backward(logits, idx, w)
        ctx.mark_non_differentiable(idx)
        return idx, w

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, grad_w):
        logits, idx, w = ctx.saved_tensors
        return ctx.layer.route_topk_grad(_whole(logits), idx, w, grad_w.contiguous()), None


class _SortRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, layer, dst_row, rows_padded, counts, pad_offsets):
        ctx.layer = layer
        ctx.save_for_backward(dst_row)
        return layer.permute_rows(x, dst_row, rows_padded, counts, pad_offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_rows):
        return ctx.layer.permute_rows_grad(_whole(grad_rows), ctx.saved_tensors[0]), None, None, None, None, None


class _CombineRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, out_rows, topk_w, shared_out, layer, dst_row, topk_idx, counts, pad_offsets):
        ctx.layer = layer
        ctx.save_for_backward(out_rows, topk_w, dst_row, counts, pad_offsets)
        return layer.combine(out_rows, dst_row, topk_idx, topk_w, shared_out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        out_rows, topk_w, dst_row, counts, pad_offsets = ctx.saved_tensors
        grad_y = _whole(grad_y)
        grows = gw = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            grows, gw = ctx.layer.combine_grad(grad_y, out_rows, dst_row, topk_w, counts, pad_offsets,
                                               need_rows=ctx.needs_input_grad[0], need_w=ctx.needs_input_grad[1])
        return grows, gw, grad_y if ctx.needs_input_grad[2] else None, None, None, None, None, None


def route(layer: MoELayer, logits: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """MoELayer.route_topk, its weights differentiable in the logits (the picks are constants)."""
    return _Route.apply(logits, layer)


def sort_rows(layer: MoELayer, x: torch.Tensor, dst_row: torch.Tensor, rows_padded: int, counts: torch.Tensor,
              pad_offsets: torch.Tensor) -> torch.Tensor:
    """MoELayer.permute_rows by a plan of distinct experts per token, differentiable in x."""
    return _SortRows.apply(x, layer, dst_row, rows_padded, counts, pad_offsets)


def combine_rows(layer: MoELayer, out_rows: torch.Tensor, dst_row: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor,
                 counts: torch.Tensor, pad_offsets: torch.Tensor, shared_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """MoELayer.combine, differentiable in out_rows, topk_w and shared_out (its bf16 modes' roundings count as the identity)."""
    return _CombineRows.apply(out_rows, topk_w, shared_out, layer, dst_row, topk_idx, counts, pad_offsets)
