"""The autograd functions of layer norm, rotary positions and attention between levels (operators the reference does not
have).  Like the convolutions' functions they ask the gradient ops for exactly the groups autograd needs, and a forward
pass that no backward pass can follow keeps nothing."""
import torch
from torch.autograd.function import once_differentiable

from .. import pccnn_lib_ops as _ops
from .convolutions import ConvFunction, keeps_projection


def _dense_rows(upstream):
    """Upstream gradients may come expanded (the gradient of a sum); the ops take rows whose values lie side by side."""
    if upstream.shape[-1] <= 1 or upstream.stride(-1) == 1:
        return upstream
    return upstream.contiguous()


class ComputeLayerNorm(ConvFunction):
    """apply(features, gamma, beta, eps) -> [N, C]: layer norm of every row (``pccnn_lib_ops.layer_norm``).  Gradients go
    to (features, gamma, beta, -)."""

    @staticmethod
    def forward(ctx, features, gamma, beta, eps):
        if not keeps_projection(ctx):
            return _ops.layer_norm(features, gamma, beta, eps)
        out, stats = _ops.layer_norm(features, gamma, beta, eps, return_stats=True)
        ctx.save_for_backward(features, gamma, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        features, gamma, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        wanted = (_ops.GRAD_FEATS if need[0] else 0) | (_ops.GRAD_WEIGHTS if need[1] or need[2] else 0)
        d_features, d_gamma, d_beta = _ops.layer_norm_grads(features, gamma, stats, _dense_rows(upstream), grad_mask=wanted)
        return d_features, d_gamma if need[1] else None, d_beta if need[2] else None, None


class ComputeRotary(ConvFunction):
    """apply(features, pts, freqs, axes, adjacent) -> [N, H, W]: pairs of features turned by pts[:, axes] * freqs
    (``pccnn_lib_ops.rotary``).  Gradients go to (features, pts, -, -, -)."""

    @staticmethod
    def forward(ctx, features, pts, freqs, axes, adjacent):
        if keeps_projection(ctx):
            ctx.adjacent_ = bool(adjacent)
            # (the gradient of the features needs the positions alone; the positions' needs the features too)
            ctx.save_for_backward(features if ctx.needs_input_grad[1] else None, pts, freqs, axes)
        return _ops.rotary(features, pts, freqs, axes, adjacent)

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        features, pts, freqs, axes = ctx.saved_tensors
        upstream = _dense_rows(upstream)
        need = ctx.needs_input_grad
        wanted = (_ops.GRAD_FEATS if need[0] else 0) | (_ops.GRAD_PTS if need[1] else 0)
        d_features, d_pts = _ops.rotary_grads(upstream if features is None else features, pts, freqs, axes, upstream,
                                              adjacent=ctx.adjacent_, grad_mask=wanted)
        return d_features, d_pts, None, None, None


class ComputeCrossAttention(ConvFunction):
    """apply(queries, keys, values, query_starts, key_starts, max_queries, max_keys, key_mask, scale) -> [M, H, W]: softmax
    attention, cloud by cloud (``pccnn_lib_ops.cross_attention``).  Gradients go to (queries, keys, values, -, ...)."""

    @staticmethod
    def forward(ctx, queries, keys, values, query_starts, key_starts, max_queries, max_keys, key_mask, scale):
        plan = (query_starts, key_starts, max_queries, max_keys)
        if not keeps_projection(ctx):
            return _ops.cross_attention(queries, keys, values, *plan, key_mask=key_mask, scale=scale)
        out, lse = _ops.cross_attention(queries, keys, values, *plan, key_mask=key_mask, scale=scale, return_lse=True)
        ctx.sizes_ = (max_queries, max_keys, scale)
        ctx.save_for_backward(queries, keys, values, query_starts, key_starts, key_mask, out, lse)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        queries, keys, values, query_starts, key_starts, key_mask, out, lse = ctx.saved_tensors
        max_queries, max_keys, scale = ctx.sizes_
        need = ctx.needs_input_grad
        wanted = (_ops.GRAD_QUERIES if need[0] else 0) | (_ops.GRAD_KEYS if need[1] or need[2] else 0)
        d_queries, d_keys, d_values = _ops.cross_attention_grads(
            queries, keys, values, query_starts, key_starts, max_queries, max_keys, out, lse, _dense_rows(upstream),
            key_mask=key_mask, scale=scale, grad_mask=wanted)
        return (d_queries, d_keys if need[1] else None, d_values if need[2] else None) + (None,) * 6
