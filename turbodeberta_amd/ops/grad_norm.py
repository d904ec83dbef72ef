"""The norm of many gradients together, and clipping by it, without a synchronisation: a launch for each 176 tensors and one for the norm, and a launch for each 128 tensors to
clip.  The device work goes through ``tdb_grads_norm`` and ``tdb_grads_clip`` (include/tdb_train.h)."""
from __future__ import annotations

import ctypes as C
import math
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from .. import _lib
from . import _launch as L

_NORMS = {2.0: 2, 1.0: 1, math.inf: 0}


def _norm_code(norm_type) -> int:
    try:
        return _NORMS[float(norm_type)]
    except (KeyError, TypeError, ValueError):
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type!r}") from None


def _max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm


def _checked(tensors: Sequence[torch.Tensor], name: str) -> None:
    for t in tensors:
        if type(t) not in (torch.Tensor, torch.nn.Parameter) or t.layout != torch.strided:
            raise ValueError(f"{name} must be dense tensors, got {type(t).__name__}" + (f" of layout {t.layout}" if torch.is_tensor(t) else ""))
    L.require_gpu(*tensors)
    for t in tensors:
        L.dtype_code(t)


def _dense(t: torch.Tensor) -> bool:
    """Values back to back in memory, in whatever order of dimensions."""
    return torch.ops.aten.is_non_overlapping_and_dense(t)


def _arguments(grads, norm: int):
    """The C ABI's arguments, with the norm's result, and all that they point to."""
    n = len(grads)
    a = _lib.GradsArgs()
    arrays = ((C.c_void_p * n)(*(t.data_ptr() for t in grads)), (C.c_int64 * n)(*(t.numel() for t in grads)), (C.c_int32 * n)(*(L.dtype_code(t) for t in grads)))
    a.tensors, a.norm = n, norm
    setattr(a, "from", C.addressof(arrays[0]))
    a.numel, a.from_dtype = C.addressof(arrays[1]), C.addressof(arrays[2])
    total = torch.empty((), dtype=torch.float32, device=grads[0].device)
    work = torch.empty(_lib.load().tdb_grads_workspace(C.byref(a)) // 8, dtype=torch.float64, device=grads[0].device)
    a.total, a.workspace, a.workspace_bytes = total.data_ptr(), work.data_ptr(), 8 * work.numel()
    return a, total, (arrays, work, grads)


def _norm(grads, norm: int):
    a, total, keep = _arguments(grads, norm)
    L.call(_lib.load().tdb_grads_norm, grads[0].device, C.byref(a))
    return a, total, keep


def _clip(a: _lib.GradsArgs, out, max_norm: float, dev) -> None:
    n = len(out)
    to, kinds = (C.c_void_p * n)(*(t.data_ptr() for t in out)), (C.c_int32 * n)(*(L.dtype_code(t) for t in out))
    a.to, a.to_dtype, a.max_norm = C.addressof(to), C.addressof(kinds), max_norm
    L.call(_lib.load().tdb_grads_clip, dev, C.byref(a))


def _scaled(grads, out, max_norm: float, norm: int, error_if_nonfinite: bool) -> torch.Tensor:
    """The norm; out = grads * factor.  What does not lie back to back, or not in the same order on both sides, goes through copies."""
    flat, to = [], []
    for t, o in zip(grads, out):
        if _dense(t) and _dense(o) and t.stride() == o.stride() and t.is_neg() == o.is_neg():       # the same place in memory is the same value on both sides
            flat.append(t), to.append(o)
        else:                                                           # by way of contiguous ones, on either side that is not
            flat.append(t.resolve_neg().contiguous())
            to.append(o if o is not t and o.is_contiguous() and not o.is_neg() else torch.empty(o.shape, dtype=o.dtype, device=o.device))
    a, total, keep = _norm(flat, norm)
    if error_if_nonfinite and not bool(torch.isfinite(total)):
        raise RuntimeError(f"the norm of the gradients is {total.item()}: nothing is clipped")
    _clip(a, to, max_norm, grads[0].device)
    for o, t in zip(out, to):
        if o is not t:
            o.copy_(t)
        elif not o.is_inference():
            torch.autograd.graph.increment_version(o)
    return total


@torch.no_grad()
def grad_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all values of all tensors together: 2 (square root of the sum of squares), 1 or ``inf``; a float32 tensor without dimensions on their device.

    tensors : one or more, float32, bfloat16 or float16 in any mix, any shapes and strides, on one device.  (None at all: 0, on the CPU.)

    Sums are held in 64 bits and added up in a fixed order: no overflow below the result's own, the same bits every time.  NaN where a value is NaN.  Not differentiable."""
    norm = _norm_code(norm_type)
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    if not tensors:
        return torch.zeros(())
    total = _lib.host().train_grads_norm(tensors, norm)
    if total is not None:
        return total
    _checked(tensors, "tensors")
    return _norm([t if _dense(t) else t.contiguous() for t in tensors], norm)[1]


@torch.no_grad()
def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0, out: Optional[Sequence[torch.Tensor]] = None,
               error_if_nonfinite: bool = False) -> Tuple[torch.Tensor, List[torch.Tensor]]:
    """``(norm, out)`` with ``norm = grad_norm(grads, norm_type)`` and ``out[i] = grads[i] * min(1, max_norm / (norm + 1e-6))``, computed in float32.

    out : tensors of the gradients' shapes, float32, bfloat16 or float16 (the float32 gradients of an optimizer, say), or the gradients themselves.  None: new ones like the
        gradients.  They must not overlap each other or another gradient.  What lies back to back in memory in the same order on both sides is read and written once, the rest is copied.
    error_if_nonfinite : raises RuntimeError, before anything is written, where the norm is infinite or NaN; that waits for the device, which nothing else here does.
        Without it a norm of NaN makes everything NaN, an infinite one 0 and NaN.

    A tensor that is its own result is not written where the factor is 1."""
    norm, max_norm = _norm_code(norm_type), _max_norm(max_norm)
    grads = list(grads)
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"out must have a tensor for each of the {len(grads)} gradients, got {len(out)}")
    if not grads:
        return torch.zeros(()), []
    if not error_if_nonfinite and out is not None:
        total = _lib.host().train_grads_clip(grads, out, norm, max_norm)
        if total is not None:
            return total, out
    _checked(grads, "gradients")
    if out is None:
        out = [torch.empty_like(t) for t in grads]
    _checked(grads[:1] + list(out), "out")
    for o, t in zip(out, grads):
        if o.shape != t.shape:
            raise ValueError(f"out must have the gradients' shapes: {tuple(o.shape)}, {tuple(t.shape)}")
        if o.is_inference() and not torch.is_inference_mode_enabled():
            raise ValueError("inference tensors cannot be written outside of inference mode")
    return _scaled(grads, out, max_norm, norm, error_if_nonfinite), out


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_``: the norm of the parameters' gradients together, which are multiplied in place by ``min(1, max_norm / (norm + 1e-6))``.

    A parameter that comes more than once counts once.  Returns the norm as ``grad_norm`` does; the rest as in ``clip_grads``."""
    parameters = [parameters] if torch.is_tensor(parameters) else parameters
    seen, grads = set(), []
    for p in parameters:
        if p.grad is not None and id(p) not in seen:
            seen.add(id(p))
            grads.append(p.grad)
    return clip_grads(grads, max_norm, norm_type, grads, error_if_nonfinite)[0]
