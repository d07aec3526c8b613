"""Differentiable forms of the layer's steps around the experts, for what is trained while the experts stay as they are: a
router calibrated behind quantising them, adapters on the expert-sorted rows.  Each is a torch.autograd.Function over the
layer's own kernels, forward and backward.  The reference has no training path (DeepseekV3MoE.forward runs moe_infer only,
modeling_deepseek_v3.py:614-626).

    idx, w = route(layer, logits)                                # w is differentiable in logits
    counts, _, pad, dst = layer.permute_plan(idx)
    rows = sort_rows(layer, x, dst, layer.padded_rows(idx.numel()), counts, pad)
    ...                                                          # experts, adapters on rows
    y = combine_rows(layer, out_rows, dst, idx, w, counts, pad, shared_out)

    h, y = add_norm(layer, x, residual, weight, eps)             # the norm in front of the block, and the residual stream
    out_rows = adapt_rows(layer, out_rows, rows, down, up, layer.adapter_plan_sorted(counts, pad, rows.shape[0]), scale)

A step can be captured into a CUDA graph, its backward pass too; as with any torch step, no eager graph of the same leaves may be alive
then (torch's accumulation nodes belong to the stream that they were made on).
"""
from typing import Optional, Tuple, Union

import torch

from . import lib as L
from .layer import AdapterPlan, MoELayer, _whole


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


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, layer, eps):
        y, h = layer.add_rmsnorm(x, residual, weight, eps)
        if residual is None:
            h = x.clone()               # an output of its own: what is done to it in place is not done to x
        ctx.layer, ctx.eps = layer, eps
        ctx.save_for_backward(x if residual is None else h, weight)
        ctx.set_materialize_grads(False)
        return h, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_h, grad_y):
        h, weight = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[0] or ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        gw = None
        if grad_y is None:
            gx = grad_h
        else:
            gx, gw = ctx.layer.add_rmsnorm_grad(grad_y.contiguous(), h, weight, ctx.eps, None if grad_h is None else grad_h.contiguous(),
                                                need_x, need_w)
            gw = None if gw is None else gw.to(weight.dtype)
        return gx if ctx.needs_input_grad[0] else None, gx if ctx.needs_input_grad[1] else None, gw, None, None


class _AdaptRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, down, up, layer, plan, scale):
        out, s = layer.adapter_add(y, x, down, up, plan, scale, keep=True)
        ctx.layer, ctx.plan = layer, plan
        ctx.scale, kept = (None, (scale,)) if isinstance(scale, torch.Tensor) else (scale, ())
        ctx.save_for_backward(x, down, up, s, *kept)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        x, down, up, s, *kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        gx = gdown = gup = None
        if any(need[1:4]):
            n_out = grad_out.shape[1]
            rows = _whole(grad_out)
            if n_out % 8:               # rows on 16-byte boundaries
                rows = torch.empty_strided(grad_out.shape, ((n_out + 7) // 8 * 8, 1), dtype=grad_out.dtype, device=grad_out.device)
                rows.copy_(grad_out)
            gx, gdown, gup = ctx.layer.adapter_grad(rows, x, down, up, ctx.plan, kept[0] if kept else ctx.scale, s, *need[1:4])
        return grad_out if need[0] else None, gx, gdown, gup, None, None, None


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


def add_norm(layer: MoELayer, x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
             eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """MoELayer.add_rmsnorm -> (h, y), differentiable in x, residual and weight: h = x + residual goes on as the residual stream, y is its
    norm.  Without a residual h is a copy of x.  At most 16384 columns where a gradient is to be taken."""
    if weight.numel() > L.NORM_GRAD_COLS and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise ValueError(f"rows of {weight.numel()}: the norm's gradient takes at most {L.NORM_GRAD_COLS} columns")
    return _AddNorm.apply(x, residual, weight, layer, eps)


def adapt_rows(layer: MoELayer, y: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, plan: AdapterPlan,
               scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """MoELayer.adapter_add by a plan, differentiable in y, x, down and up (the scales are constants)."""
    if not isinstance(plan, AdapterPlan):
        raise ValueError("adapt_rows takes a plan (adapter_plan, adapter_plan_sorted): ids could change before the gradient is taken")
    if isinstance(scale, torch.Tensor) and scale.requires_grad:
        raise ValueError("adapt_rows has no gradient for its scales: detach them")
    return _AdaptRows.apply(y, x, down, up, layer, plan, scale)
