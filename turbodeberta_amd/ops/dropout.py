"""Dropout whose mask is a function of a seed: nothing is stored for the backward pass but the seed.

The device work is one launch each way through ``tdb_dropout`` (include/tdb_train.h)."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import _launch as L


def _launch(x: torch.Tensor, threshold: int, seed: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    y = torch.empty_like(x)
    L.call(_lib.load().tdb_dropout, x.device, x.data_ptr(), y.data_ptr(), x.numel(), L.dtype_code(x), threshold, seed.data_ptr())
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, threshold, seed):
        ctx.save_for_backward(seed)
        ctx.threshold = threshold
        return _launch(x, threshold, seed)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _lib.host().backward_begins()
        return _launch(dy, ctx.threshold, *ctx.saved_tensors), None, None


def dropout(x: torch.Tensor, p: float, seed: torch.Tensor) -> torch.Tensor:
    """``x`` with values dropped with probability ``p``, the others multiplied by ``1 / (1 - p)``; ``p`` counts in units of 2^-16.

    x : float32, bfloat16 or float16, any shape and strides; the result is contiguous.  (``p`` below 2^-17: ``x`` itself.)
    seed : int64 tensor with one element on x's device; it is read when the kernel runs, so a captured graph drops other values after it has
        been changed.  The same seed, ``p`` and number of elements give the same mask.  It must not be changed between the forward and the
        backward pass (autograd raises).  Draw a new one for every call, e.g. with ``new_seed``.

    A dropped value is 0 whatever it was, infinities and NaN included.  Differentiable once."""
    y = _lib.host().train_dropout(x, p, seed)
    if y is not None:
        return y
    threshold = L.drop_threshold(p)
    L.require_gpu(x, L.one_seed(seed))
    L.dtype_code(x)
    return _Dropout.apply(x, threshold, seed) if threshold else x


def new_seed(device) -> torch.Tensor:
    """A seed from PyTorch's generator of the device (its state and ``torch.manual_seed`` decide; also under graph capture)."""
    return torch.empty(1, dtype=torch.int64, device=device).random_()
