"""Softmax cross entropy over a vocabulary, from hidden states and the output layer, with its gradient, as masked language modelling has it
(modeling_deberta_v2.py: DebertaV2ForMaskedLM).

The logits, rows x vocabulary, are never in memory.  The device work goes through ``tdb_loss_fwd`` and ``tdb_loss_bwd`` (include/tdb_train.h)."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import _launch as L

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """``[rows, hidden]``, columns side by side; a view where there is one."""
    x = x.resolve_neg().reshape(-1, x.shape[-1])
    return x if (x.shape[1] == 1 or x.stride(1) == 1) and x.stride(0) >= 0 else x.contiguous()


def _weight_rows(w: torch.Tensor) -> torch.Tensor:
    """Rows that the kernels can address: values side by side, at multiples of 4 bytes; a copy where they are not."""
    w, es = w.resolve_neg(), w.element_size()
    apart = w.shape[1] if w.shape[0] == 1 else w.stride(0)
    if (w.shape[1] == 1 or w.stride(1) == 1) and w.data_ptr() % 4 == 0 and w.shape[1] <= apart and (apart * es) % 4 == 0 and apart * es <= 1 << 22:
        return w
    if (w.shape[1] * es) % 4 == 0:
        return L.copied(w)
    return torch.empty(w.shape[0], w.shape[1] + 1, dtype=w.dtype, device=w.device)[:, :-1].copy_(w)


def _arguments(weight, bias, rows, hidden, ignore_index, reduction) -> _lib.LossArgs:
    a = _lib.LossArgs()
    a.dtype, a.bias_dtype = L.dtype_code(weight), L.dtype_code(weight if bias is None else bias)
    a.hidden, a.reduction, a.rows, a.vocab, a.ignore_index = hidden, reduction, rows, weight.shape[0], ignore_index
    a.weight, a.weight_stride, a.bias = weight.data_ptr(), hidden + 3 & ~3 if weight.shape[0] == 1 else weight.stride(0), None if bias is None else bias.data_ptr()
    return a


def _call(fn, a: _lib.LossArgs, state: torch.Tensor, backward: int) -> None:
    a.state, a.state_bytes = state.data_ptr(), state.numel()
    work = torch.empty(_lib.load().tdb_loss_workspace(C.byref(a), backward), dtype=torch.uint8, device=state.device)
    a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
    L.call(fn, state.device, C.byref(a))


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, labels, bias, ignore_index, reduction):
        rows, w, b, y = _as_rows(x), _weight_rows(weight), None if bias is None else bias.resolve_neg().contiguous(), labels.resolve_neg().contiguous()
        loss = torch.empty(labels.shape if reduction == 0 else (), dtype=torch.float32, device=x.device)
        a = _arguments(w, b, labels.numel(), x.shape[-1], ignore_index, reduction)
        a.x, a.x_stride, a.labels, a.loss = rows.data_ptr(), rows.stride(0), y.data_ptr(), loss.data_ptr()
        state = torch.empty(_lib.load().tdb_loss_state(C.byref(a)), dtype=torch.uint8, device=x.device)
        _call(_lib.load().tdb_loss_fwd, a, state, 0)
        ctx.save_for_backward(weight, bias, state)
        ctx.shape, ctx.ignore_index, ctx.reduction, ctx.rows = x.shape, ignore_index, reduction, labels.numel()
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        _lib.host().backward_begins()
        weight, bias, state = ctx.saved_tensors
        w, b = _weight_rows(weight), None if bias is None else bias.resolve_neg().contiguous()
        hidden = ctx.shape[-1]
        a = _arguments(w, b, ctx.rows, hidden, ctx.ignore_index, ctx.reduction)
        dloss = dloss.float().resolve_neg()
        if ctx.reduction == 0:
            dloss = dloss.reshape(-1)
            if dloss.numel() > 1 and dloss.stride(0) < 0:
                dloss = dloss.contiguous()
        a.dloss, a.dloss_stride = dloss.data_ptr(), dloss.stride(0) if dloss.dim() else 0
        want_x, want_w, _, want_b = ctx.needs_input_grad[:4]
        dx = torch.empty(ctx.shape, dtype=weight.dtype, device=weight.device) if want_x else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if want_w else None
        db = torch.empty(bias.shape, dtype=bias.dtype, device=weight.device) if bias is not None and want_b else None
        a.dx, a.dweight, a.dbias = (None if t is None else t.data_ptr() for t in (dx, dw, db))
        a.dx_stride = a.dweight_stride = hidden
        _call(_lib.load().tdb_loss_bwd, a, state, 1)
        return dx, dw, None, db, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, bias: Optional[torch.Tensor] = None, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """``torch.nn.functional.cross_entropy(x @ weight.T + bias, labels, ignore_index=.., reduction=..)`` in float32, without the logits in memory.

    x : float32, bfloat16 or float16 ``[.., hidden]``, hidden up to 32768, any strides.
    weight : ``[vocab, hidden]`` in x's dtype.  bias : ``[vocab]`` in x's dtype or float32, or None.
    labels : int64 of x's shape without the last dimension.  Rows with ``ignore_index`` do not count: nothing of them is read or computed, and their loss and gradient are 0.
        A label outside ``[0, vocab)`` makes its row's loss NaN, and with it a sum or mean and the gradients that the row goes into.
    reduction : "mean" over the rows that count (NaN if there are none), "sum", or "none": a loss for each row.

    The loss is float32.  Sums are held in float32 or more and added up in a fixed order; the gradient of the logits is rounded to x's dtype for the matrix instructions
    (in float16 scaled, so that probabilities down to 2^-38 count), which adds up to 40 % to the error that rounded results have.  Differentiable once, with respect to x, weight and bias."""
    loss = _lib.host().train_loss(x, weight, labels, bias, ignore_index, _REDUCTIONS.get(reduction))
    if loss is not None:
        return loss
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if not all(torch.is_tensor(t) for t in (x, weight, labels)) or not (bias is None or torch.is_tensor(bias)):
        raise ValueError("x, weight, labels and bias must be tensors")
    L.require_gpu(x, weight, labels, bias)
    L.dtype_code(x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 32768:
        raise ValueError(f"x must have rows of 1 to 32768 values, got {tuple(x.shape)}")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or not 1 <= weight.shape[0] <= 1 << 27 or weight.dtype != x.dtype:
        raise ValueError(f"weight must be [vocab, {x.shape[-1]}] of {x.dtype}, got {tuple(weight.shape)} {weight.dtype}")
    if labels.dtype != torch.int64 or labels.shape != x.shape[:-1] or labels.numel() > 1 << 27:
        raise ValueError(f"labels must be int64 {tuple(x.shape[:-1])}, got {tuple(labels.shape)} {labels.dtype}")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f"bias must be [{weight.shape[0]}] of {x.dtype} or float32, got {tuple(bias.shape)} {bias.dtype}")
    if not isinstance(ignore_index, int) or isinstance(ignore_index, bool) or not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index must be a 64-bit integer, got {ignore_index!r}")
    return _Loss.apply(x, weight, labels, bias, ignore_index, _REDUCTIONS[reduction])
