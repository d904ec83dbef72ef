"""LayerNorm with its backward pass, by itself and behind dropout and a residual, as DeBERTa's layers have it.

The device work is one launch forward and two backward (the second adds up the weight's and bias's gradient in a fixed order), through
``tdb_norm_fwd`` and ``tdb_norm_bwd`` (include/tdb_train.h)."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import _launch as L


def _as_rows(t: torch.Tensor, hidden: int) -> torch.Tensor:
    """``[rows, hidden]``, columns side by side; a view where there is one."""
    t = t.reshape(-1, hidden)
    return t if hidden == 1 or t.stride(1) == 1 else t.contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, threshold, seed, eps):
        hidden = x.shape[-1]
        rows, res = _as_rows(x, hidden), None if residual is None else _as_rows(residual, hidden)
        w, b = (None, None) if weight is None else (weight.contiguous(), bias.contiguous())
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a = _lib.NormArgs(L.dtype_code(x), L.dtype_code(x if w is None else w), hidden, threshold, rows.shape[0], eps, 0, rows.data_ptr(), _ptr(res), _ptr(w),
                          _ptr(b), None, y.data_ptr(), None, None, None, None, None, _ptr(seed), rows.stride(0), 0 if res is None else res.stride(0),
                          0, hidden, 0, 0)
        L.call(_lib.load().tdb_norm_fwd, x.device, C.byref(a))
        ctx.save_for_backward(x, residual, weight, bias, seed)
        ctx.threshold, ctx.eps = threshold, eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _lib.host().backward_begins()
        x, residual, weight, bias, seed = ctx.saved_tensors
        want_x, want_res, want_w, want_b = ctx.needs_input_grad[:4]
        hidden = x.shape[-1]
        rows, res, dy = _as_rows(x, hidden), None if residual is None else _as_rows(residual, hidden), _as_rows(dy, hidden)
        w, b = (None, None) if weight is None else (weight.contiguous(), bias.contiguous())
        new = lambda like: torch.empty(like.shape, dtype=like.dtype, device=x.device)
        dx = new(x) if want_x else None
        dres = new(residual) if want_res else None
        dw = db = work = None
        lib = _lib.load()
        if want_w or want_b:
            dw, db = new(weight), new(bias)
            work = torch.empty(lib.tdb_norm_workspace(rows.shape[0], hidden), dtype=torch.float32, device=x.device)
        a = _lib.NormArgs(L.dtype_code(x), L.dtype_code(x if w is None else w), hidden, ctx.threshold, rows.shape[0], ctx.eps, 0, rows.data_ptr(), _ptr(res),
                          _ptr(w), _ptr(b), dy.data_ptr(), None, _ptr(dx), _ptr(dres), _ptr(dw), _ptr(db), _ptr(work), _ptr(seed), rows.stride(0),
                          0 if res is None else res.stride(0), dy.stride(0), 0, hidden, hidden)
        L.call(lib.tdb_norm_bwd, x.device, C.byref(a))
        return dx, dres, dw if want_w else None, db if want_b else None, None, None, None


def _norm(x, residual, weight, bias, threshold, seed, eps):
    dev = L.require_gpu(x, residual, weight, bias, seed)
    L.dtype_code(x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 32768:
        raise ValueError(f"x must have rows of 1 to 32768 values, got {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must have the shape and dtype of x: {tuple(residual.shape)} {residual.dtype}, {tuple(x.shape)} {x.dtype}")
    if (weight is None) != (bias is None):
        raise ValueError("weight and bias: both or neither")
    if weight is not None:
        if weight.shape != x.shape[-1:] or bias.shape != x.shape[-1:]:
            raise ValueError(f"weight and bias must be [{x.shape[-1]}], got {tuple(weight.shape)} and {tuple(bias.shape)}")
        if weight.dtype != bias.dtype or weight.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"weight and bias must both have the dtype of x or float32, got {weight.dtype} and {bias.dtype}")
    eps = float(eps)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    return _Norm.apply(x, residual, weight, bias, threshold, seed, eps)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-7) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension; contiguous result of x's shape and dtype.

    x : float32, bfloat16 or float16 ``[.., hidden]``, hidden up to 32768, any strides.
    weight, bias : ``[hidden]``, both or neither, in x's dtype or float32.

    Statistics, sums and the gradient of weight and bias are held in float32; the latter is added up in a fixed order.  Differentiable once."""
    y = _lib.host().train_norm(x, None, weight, bias, 0, None, eps)
    return _norm(x, None, weight, bias, 0, None, eps) if y is None else y


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                           p: float = 0.0, seed: Optional[torch.Tensor] = None, eps: float = 1e-7) -> torch.Tensor:
    """``layer_norm(dropout(x, p, seed) + residual, weight, bias, eps)`` in one pass over x and residual, which the backward pass reads again
    instead of what lies between (modeling_deberta_v2.py:42-53, :400-411).  x and residual have one shape and dtype; the
    rest as in ``layer_norm`` and ``ops.dropout.dropout``, whose mask for x this is."""
    if residual is None:
        raise ValueError("residual is required: layer_norm takes rows without one")
    y = _lib.host().train_norm(x, residual, weight, bias, p, seed, eps)
    if y is not None:
        return y
    threshold = L.drop_threshold(p)
    return _norm(x, residual, weight, bias, threshold, L.one_seed(seed) if threshold else None, eps)
