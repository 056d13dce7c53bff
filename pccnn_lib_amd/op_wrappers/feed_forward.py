"""The autograd functions of the root-mean-square norm and the gated linear map (operators the reference does not have)."""
import torch
from torch.autograd.function import once_differentiable

from .. import pccnn_lib_ops as _ops
from .attention import _dense_rows
from .convolutions import ConvFunction, keeps_projection


class ComputeRMSNorm(ConvFunction):
    """apply(features, gamma, residual, eps) -> [N, C]: root-mean-square norm of every row (``pccnn_lib_ops.rms_norm``); with a
    residual (or None) of features + residual, whose sum comes back too.  Gradients go to (features, gamma, residual, -)."""

    @staticmethod
    def forward(ctx, features, gamma, residual, eps):
        if not keeps_projection(ctx):
            return _ops.rms_norm(features, gamma, residual, eps)
        ctx.set_materialize_grads(False)            # (a result that nobody uses has no gradient, not one of zeros)
        results = _ops.rms_norm(features, gamma, residual, eps, return_stats=True)
        total = features if residual is None else results[1]
        ctx.save_for_backward(total, gamma, results[-1])
        return results[0] if residual is None else results[:2]

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream, total_upstream=None):
        total, gamma, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        if upstream is None:
            return total_upstream if need[0] else None, None, total_upstream if need[2] else None, None
        wanted = (_ops.GRAD_FEATS if need[0] or need[2] else 0) | (_ops.GRAD_WEIGHTS if need[1] else 0)
        d_features, d_gamma = _ops.rms_norm_grads(total, gamma, rstd, _dense_rows(upstream),
                                                  None if total_upstream is None else _dense_rows(total_upstream),
                                                  grad_mask=wanted)
        return d_features if need[0] else None, d_gamma, d_features if need[2] else None, None


class ComputeGatedLinear(ConvFunction):
    """apply(features, gate, up, activation) -> [N, H]: act(features gate^T) * (features up^T) (``pccnn_lib_ops.gated_linear``).
    Keeps its inputs alone; the backward pass forms both projections anew.  Gradients go to (features, gate, up, -)."""

    @staticmethod
    def forward(ctx, features, gate, up, activation):
        if keeps_projection(ctx):
            ctx.activation_ = activation
            ctx.save_for_backward(features, gate, up)
        return _ops.gated_linear(features, gate, up, activation)

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        features, gate, up = ctx.saved_tensors
        need = ctx.needs_input_grad
        wanted = (_ops.GRAD_FEATS if need[0] else 0) | (_ops.GRAD_WEIGHTS if need[1] or need[2] else 0)
        d_features, d_gate, d_up = _ops.gated_linear_grads(features, gate, up, _dense_rows(upstream), ctx.activation_,
                                                           grad_mask=wanted)
        return d_features, d_gate if need[1] else None, d_up if need[2] else None, None
