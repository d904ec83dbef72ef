"""Modules of a DeBERTa-v2/v3 model that is trained with this package's operators.

``patch_model(model, training=True)`` (``turbodeberta_amd.model``) switches a model's dropouts, LayerNorms and output blocks to the classes below and
its attention to ``ops.trainable_attention``.  They add no parameters and no state.  In training mode, and in evaluation where autograd records, they
call the operators for tensors on the GPU in float32, bfloat16 or float16, which store no masks, no probabilities and nothing between
dropout, residual and LayerNorm; everything else -- evaluation under ``torch.no_grad``, the CPU -- runs the parent class's code.

An operator that takes the place of several modules runs none of them, so it does so only where they are what their classes say: a dropout or LayerNorm
that has been replaced by another class's, or that has hooks or a ``forward`` of its own, is called (``stands_for``).

Training mode under ``torch.no_grad`` counts as well: checkpointing of the reentrant kind runs a layer that way first and again with gradients, and
both runs have to draw the same masks."""
from __future__ import annotations

import torch
from torch import nn
from transformers.models.deberta_v2.modeling_deberta_v2 import DebertaV2Output, DebertaV2SelfOutput

from .ops.dropout import dropout, new_seed
from .ops.layer_norm import dropout_add_layer_norm, layer_norm

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def operators_take(module: nn.Module, *tensors) -> bool:
    """Whether a module's call with these tensors is one for the training operators."""
    return (module.training or torch.is_grad_enabled()) and all(t.is_cuda and t.dtype in _TYPES for t in tensors)


def draw_seed(module: nn.Module, device) -> torch.Tensor:
    """The seed of a module's next dropout, from PyTorch's generator of the device: ``torch.manual_seed`` decides, and gradient checkpointing, which
    puts the generator's state back, finds the same masks."""
    return new_seed(device)


def stands_for(module: nn.Module, *classes) -> bool:
    """Whether an operator may stand for a call of ``module``: it is one of these classes and no subclass, with the ``forward`` that the class had when this
    file was imported, and nobody watches the call."""
    return (type(module) in classes and type(module).forward is _FORWARDS[type(module)] and "forward" not in module.__dict__ and module._compiled_call_impl is None
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks)
            and not torch.nn.modules.module._has_any_global_hook())


def is_dropout(drop: nn.Module) -> bool:
    """Whether ``rate_of`` says all about a dropout: a stock one, or none (``nn.Identity``)."""
    return stands_for(drop, nn.Dropout, FlashDropout, nn.Identity)


def rate_of(module: nn.Module, drop: nn.Module) -> float:
    """The probability that ``drop``, a dropout of ``module``, drops a value with in the next call."""
    return float(drop.p) if isinstance(drop, nn.Dropout) and drop.training else 0.0


class FlashDropout(nn.Dropout):
    """``nn.Dropout`` by ``ops.dropout.dropout``."""

    def forward(self, x):
        if not (self.training and self.p > 0 and not self.inplace and operators_take(self, x)):
            return super().forward(x)
        return dropout(x, self.p, draw_seed(self, x.device))


def _norm_arguments(norm: nn.LayerNorm, x):
    """``(x, weight, bias)`` of a call of the norm's operators; None where they do not take it.  Autocast has LayerNorm computed in float32."""
    if torch.is_autocast_enabled("cuda"):
        x = x.float()
    w, b = norm.weight, norm.bias
    if tuple(norm.normalized_shape) != tuple(x.shape[-1:]) or (w is None) != (b is None) or x.shape[-1] > 32768:
        return None
    if w is not None and (w.dtype != b.dtype or w.dtype not in (x.dtype, torch.float32)):
        return None
    return x, w, b


class FlashLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` by ``ops.layer_norm.layer_norm``."""

    def forward(self, x):
        a = _norm_arguments(self, x) if operators_take(self, x) else None
        return super().forward(x) if a is None else layer_norm(*a, self.eps)


_FORWARDS = {c: c.forward for c in (nn.Dropout, nn.Identity, nn.LayerNorm, FlashDropout, FlashLayerNorm)}


class _Output:
    """``LayerNorm(dropout(dense(x)) + input)`` (modeling_deberta_v2.py:42-53, :400-411) by ``ops.layer_norm.dropout_add_layer_norm``."""

    def forward(self, hidden_states, input_tensor):
        if not (operators_take(self, hidden_states, input_tensor) and is_dropout(self.dropout) and stands_for(self.LayerNorm, nn.LayerNorm, FlashLayerNorm)):
            return super().forward(hidden_states, input_tensor)
        x = self.dense(hidden_states)
        wide = torch.promote_types(x.dtype, input_tensor.dtype)
        a = _norm_arguments(self.LayerNorm, x.to(wide))
        if a is None or x.shape != input_tensor.shape:
            return self.LayerNorm(self.dropout(x) + input_tensor)
        x, weight, bias = a
        p = rate_of(self, self.dropout)
        return dropout_add_layer_norm(x, input_tensor.to(x.dtype), weight, bias, p, draw_seed(self, x.device) if p else None, self.LayerNorm.eps)


class FlashDebertaV2SelfOutput(_Output, DebertaV2SelfOutput):
    pass


class FlashDebertaV2Output(_Output, DebertaV2Output):
    pass
