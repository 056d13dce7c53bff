"""The feed-forward half of a block between levels (no counterpart in the reference): what follows ``CrossAttention`` on the
features of every point by itself, and its form for deployed networks in 8-bit integers."""
import torch

from ... import pccnn_lib_ops as _ops
from ...op_wrappers import ComputeGatedLinear
from .norm import RMSNormalization, of_one_type


class GatedFeedForward(torch.nn.Module):
    """Features of every point updated by themselves:

        s + down(act(gate(norm(s))) * up(norm(s))),   s = x, or x + update

    with x [N, p_num_features] and ``p_update`` [N, p_num_features] what the layer before adds to them, where it has not yet (the
    addition is part of the norm's kernel; ``CrossAttention``'s result is its features with the update added: x as it is).  ``p_hidden``: hidden channels, by default 8/3 of the features in whole eights, which makes three maps as large
    as two of four times the features.  ``p_activation``: "silu", "gelu", "sigmoid" or "relu".  Sub-modules ``norm_``
    (``RMSNormalization``), ``gate_``, ``up_``, ``down_`` (linear maps).  float32 or bfloat16 (``.to(torch.bfloat16)``); under
    autocast to bfloat16 the norm's result and the weights of all three maps are bfloat16, like those of any linear map."""

    def __init__(self, p_num_features, p_hidden=None, p_activation="silu", p_eps=1e-6):
        super(GatedFeedForward, self).__init__()
        hidden = -(-(8 * p_num_features) // 24) * 8 if p_hidden is None else int(p_hidden)
        if p_num_features < 1 or hidden < 1:
            raise RuntimeError("GatedFeedForward: %d features, %d hidden channels" % (p_num_features, hidden))
        if p_activation not in _ops.ACTIVATIONS:
            raise RuntimeError("GatedFeedForward: activation %r (%s)" % (p_activation, ", ".join(_ops.ACTIVATIONS)))
        self.num_features_, self.hidden_, self.activation_ = p_num_features, hidden, p_activation
        self.norm_ = RMSNormalization(p_num_features, p_eps)
        self.gate_ = torch.nn.Linear(p_num_features, hidden, bias=False)
        self.up_ = torch.nn.Linear(p_num_features, hidden, bias=False)
        self.down_ = torch.nn.Linear(hidden, p_num_features)

    def forward(self, p_feats, p_update=None):
        if p_update is None:
            normed, total = self.norm_(p_feats), p_feats
        else:
            normed, total = self.norm_(p_feats, p_update)
        gate, up = self.gate_.weight, self.up_.weight
        if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
            normed, gate, up = normed.to(torch.bfloat16), gate.to(torch.bfloat16), up.to(torch.bfloat16)
        return total + self.down_(ComputeGatedLinear.apply(normed, gate, up, self.activation_))


class GatedFeedForward8Bit(torch.nn.Module):
    """A ``GatedFeedForward`` on the GPU deployed in 8 bits: its weights as integers with a scale for every output channel, laid
    out here once; in a call the normed features and the hidden ones get a scale for every row.  Same arguments and results as the
    layer it is made from, float32 or bfloat16 features; no gradients.  Buffers ``gamma_``, ``{gate,up,down}_codes_``,
    ``{gate,up,down}_scales_``, ``bias_``; scales, gamma and bias stay float32 whatever type the module is moved to."""

    def __init__(self, p_layer):
        super(GatedFeedForward8Bit, self).__init__()
        self.num_features_, self.hidden_, self.activation_ = p_layer.num_features_, p_layer.hidden_, p_layer.activation_
        self.eps_ = p_layer.norm_.eps_
        # (outside inference mode, whose tensors a later training run could not share a module with)
        with torch.inference_mode(False), torch.no_grad():
            self.register_buffer("gamma_", p_layer.norm_.gamma_.detach().reshape(-1).float().clone())
            bias = p_layer.down_.bias
            self.register_buffer("bias_", None if bias is None else bias.detach().float().clone())
            for name in ("gate", "up", "down"):
                codes, scales = _ops.quantize_rows(getattr(p_layer, name + "_").weight.detach())
                self.register_buffer(name + "_codes_", codes)
                self.register_buffer(name + "_scales_", scales)

    def _apply(self, fn, *args, **kwargs):
        kept = {name: buffer for name, buffer in self.named_buffers() if buffer.is_floating_point()}
        super(GatedFeedForward8Bit, self)._apply(fn, *args, **kwargs)
        for name, buffer in kept.items():
            moved = getattr(self, name)
            if moved.dtype != buffer.dtype:
                setattr(self, name, buffer.to(moved.device))
        return self

    def forward(self, p_feats, p_update=None):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (p_feats, p_update)):
            raise RuntimeError("GatedFeedForward8Bit: no gradients (call it under torch.no_grad())")
        p_feats, p_update = of_one_type(p_feats, p_update)
        got = _ops.rms_norm_8bit(p_feats, self.gamma_, p_update, self.eps_)
        total = p_feats if p_update is None else got[2]
        hidden = _ops.gated_linear_8bit(got[0], got[1], self.gate_codes_, self.gate_scales_, self.up_codes_, self.up_scales_,
                                        self.activation_, p_feats.dtype)
        codes, scales = _ops.quantize_rows(hidden)
        return total + _ops.linear_8bit(codes, scales, self.down_codes_, self.down_scales_, self.bias_, p_feats.dtype)
