"""Disentangled attention with its gradient, for training: padded batches and packed sequences.

What ``ops.flash_attention`` and ``ops.flash_attention_varlen`` compute forward only, with dropout on the probabilities and gradients of q, k, v and
of both position tables.  No ``[L, L]`` array and no mask outlives a call: the forward pass keeps its inputs, its result, one number for each row and, in 16
bits, what rounding took from the result, as much again; the backward pass holds the scores' gradients of a few heads at a time (2 GiB, or one head
if that has more: element size x sum of length x longest), and with tables sums by relative position: up to half that size, 96 MiB, or 128 KiB for each of the
heads and 64 tokens of the longest sequence, and no more than 2 GiB unless one head has.
The device work goes through ``tdb_attn_train_fwd`` and ``tdb_attn_train_bwd`` (include/tdb_train.h)."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import _launch as L


def _strides(t):
    """(batch, head, row) strides of ``[B, H, L, D]``, or of packed ``[T, H, D]``."""
    return (t.stride(0), t.stride(1), t.stride(2)) if t.dim() == 4 else (0, t.stride(1), t.stride(0))


def _apart(t):
    """t where the kernels can address it: aligned rows that do not share memory, not too far apart for 32-bit offsets."""
    stride = t.stride(-2) if t.dim() == 4 else t.stride(0)
    return t if L.rows_ok(t) and t.shape[-1] <= stride <= (1 << 24) // t.element_size() else L.copied(t)


def _like(t):
    """A tensor for results of t's shape: t's strides where the kernels can address them, else contiguous."""
    o = torch.empty_like(t)
    return o if _apart(o) is o else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _args(q, k, v, o, rest, lse, pk, pq, lens, cu, longest, scale, buckets, max_rel, threshold, seed):
    a = _lib.TrainAttnArgs()
    packed = cu is not None
    a.dtype, a.heads, a.head_dim, a.max_seqlen, a.threshold, a.sm_scale = L.dtype_code(q), q.shape[1], q.shape[-1], longest, threshold, scale
    a.batch, a.total_tokens = (cu.numel() - 1, q.shape[0]) if packed else (q.shape[0], 0)
    _fill(a, q=q, k=k, v=v, o=o)
    a.lse = lse.data_ptr()
    if rest is not None:
        a.o_rest = rest.data_ptr()
    if packed:
        a.cu_seqlens = cu.data_ptr()
    elif lens is not None:
        a.seqlens_k = lens.data_ptr()
    if pk is not None or pq is not None:
        lut, a.lut_half = L.delta_lut(q.device, longest, buckets, max_rel)
        a.delta_lut, a.span = lut.data_ptr(), L.att_span(buckets, max_rel)
        for name, t in (("pos_key", pk), ("pos_query", pq)):
            if t is not None:
                setattr(a, name, t.data_ptr())
                setattr(a, name + "_stride_h", t.stride(0))
                setattr(a, name + "_stride_r", t.stride(1))
    if threshold:
        a.seed = seed.data_ptr()
    return a


def _fill(a, **tensors):
    for name, t in tensors.items():
        setattr(a, name, t.data_ptr())
        for axis, s in zip("bhl", _strides(t)):
            setattr(a, f"{name}_stride_{axis}", s)


def _shaped(t, shape):
    return None if t is None else t.view(shape)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, pk, pq, lens, cu, seed, *plain):
        q, k, v = _apart(q), _apart(k), _apart(v)
        ctx.shapes = [None if t is None else t.shape for t in (pk, pq)]
        # (A leading 1 is taken off in here, so that a leaf's accumulation is this node's own edge, which backward_begins looks at.)
        pk, pq = (None if t is None else L.as_rows(t[0] if t.dim() == 4 else t) for t in (pk, pq))
        o = _like(q)
        ctx.plain, ctx.nothing = plain, q.numel() == 0 or (cu is not None and cu.numel() < 2)
        if ctx.nothing:                     # no sequences, or none with a token: nothing is launched
            ctx.save_for_backward(q, k, v, pk, pq)
            return o.zero_()
        lse = torch.empty(q.shape[1], q.numel() // max(q.shape[1] * q.shape[-1], 1), dtype=torch.float32, device=q.device)
        rest = None if q.dtype == torch.float32 else torch.empty(*lse.shape, q.shape[-1], dtype=q.dtype, device=q.device)
        a = _args(q, k, v, o, rest, lse, pk, pq, lens, cu, *plain, seed)
        L.call(_lib.load().tdb_attn_train_fwd, q.device, C.byref(a))
        ctx.save_for_backward(q, k, v, o, rest, lse, pk, pq, lens, cu, seed)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        _lib.host().backward_begins()
        if ctx.nothing:
            grads = [None if t is None else torch.zeros_like(t) for t in ctx.saved_tensors]
            return (*grads[:3], *map(_shaped, grads[3:], ctx.shapes)) + (None,) * (3 + len(ctx.plain))
        q, k, v, o, rest, lse, pk, pq, lens, cu, seed = ctx.saved_tensors
        dout = _apart(dout)
        dq, dk, dv = _like(q), _like(k), _like(v)
        a = _args(q, k, v, o, rest, lse, pk, pq, lens, cu, *ctx.plain, seed)
        _fill(a, dout=dout, dq=dq, dk=dk, dv=dv)
        tables = []
        for name, t in (("dpos_key", pk), ("dpos_query", pq)):
            grad = None
            if t is not None:
                grad = (torch.empty if t.shape[1] == 2 * a.span else torch.zeros)(t.shape, dtype=t.dtype, device=t.device)
                setattr(a, name, grad.data_ptr())
                setattr(a, name + "_stride_h", grad.stride(0))
            tables.append(grad)
        lib = _lib.load()
        a.workspace_bytes = lib.tdb_attn_train_workspace(C.byref(a))
        work = torch.empty(a.workspace_bytes, dtype=torch.uint8, device=q.device)
        a.workspace = work.data_ptr()
        L.call(lib.tdb_attn_train_bwd, q.device, C.byref(a))
        return (dq, dk, dv, *map(_shaped, tables, ctx.shapes)) + (None,) * (3 + len(ctx.plain))


def _checked(q, k, v, pos_key_layer, pos_query_layer, heads, sm_scale, buckets, max_rel, p, seed, longest, reach, others):
    """(sm_scale, tables, threshold, seed) of a call whose q, k, v have been looked at by themselves.  reach: what no sequence is longer than."""
    threshold = L.drop_threshold(p)
    seed = L.one_seed(seed) if threshold else None
    L.require_gpu(q, k, v, pos_key_layer, pos_query_layer, seed, *others)
    L.dtype_code(q)
    D = q.shape[-1]
    if k.shape != q.shape or v.shape != q.shape or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("self-attention only: q, k, v must have one shape and dtype")
    if D % 8 or not 8 <= D <= 64:
        raise ValueError(f"head dimension {D}: need a multiple of 8 up to 64")
    scale = L.default_scale(sm_scale, D)
    if not 0 < scale < 1e30:
        raise ValueError("sm_scale must be positive")
    tables = []
    span = L.att_span(buckets, max_rel)
    if (pos_key_layer is not None or pos_query_layer is not None) and span < 1:
        raise ValueError("position terms need position_buckets > 0 or max_relative_distance > 0")
    for name, t in (("pos_key_layer", pos_key_layer), ("pos_query_layer", pos_query_layer)):
        if t is not None:
            if t.dtype != q.dtype:
                raise ValueError("position tables must have the dtype of q")
            shape = t.shape[1:] if t.dim() == 4 and t.shape[0] == 1 else t.shape
            if len(shape) != 3 or shape[0] != heads or shape[2] != D or shape[1] < 2 * span:
                raise ValueError(f"{name}: expected [H={heads}, >=2*span={2 * span}, D={D}], got {tuple(t.shape)}")
        tables.append(t)
    if longest <= 1 << 20 and not all(t is None for t in tables):        # (the C side refuses longer ones)
        L.require_rising(q.device, longest, reach, buckets, max_rel)
    return scale, tables, threshold, seed


def trainable_attention_with_disentangled(q, k, v, pos_key_layer: Optional[torch.Tensor] = None, pos_query_layer: Optional[torch.Tensor] = None,
                                          sm_scale: Optional[float] = None, position_buckets: int = 0, max_relative_distance: int = 0, *,
                                          seqlens_k: Optional[torch.Tensor] = None, dropout_p: float = 0.0, seed: Optional[torch.Tensor] = None):
    """``dropout(softmax(sm_scale * (Q K^T + c2p + p2c))) V`` of a padded batch, differentiable once in q, k, v and the tables.

    q, k, v : ``[B, H, L, D]``, float32, bfloat16 or float16, D a multiple of 8 up to 64; any strides with a contiguous last dimension and rows at
        multiples of 16 bytes (others are copied).  The result has q's shape and strides.
    pos_key_layer, pos_query_layer : ``[H, >= 2*span, D]`` (or with a leading 1) projections of the relative embeddings, or None; indexed as in
        ``ops.flash_attention.flash_attention_with_disentangled``, as are position_buckets and max_relative_distance.  (Buckets that run backwards, max_relative_distance - 1 <=
        position_buckets / 2, are refused beyond position_buckets / 2 + 1 tokens.)
    sm_scale : positive; None means ``1/sqrt(D)``.
    seqlens_k : int32 ``[B]`` valid lengths of right-padded sequences.  Rows beyond are zeros in the result and in every gradient; what the inputs and
        the result's gradient hold there is not read.
    dropout_p, seed : of the probabilities, as in ``ops.dropout.dropout``; the mask is a function of seed, sequence, head, query and key, so a padded and a
        packed batch of the same sequences drop the same.

    Scores, sums and the gradients' sums are held in float32; probabilities and the scores' gradients are rounded to the type where they enter a product."""
    o = _lib.host().train_attention(q, k, v, pos_key_layer, pos_query_layer, sm_scale, position_buckets, max_relative_distance, seqlens_k, None, 0, dropout_p, seed)
    if o is not None:
        return o
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must be [B, H, L, D]")
    longest = max(q.shape[2], 1)
    scale, (pk, pq), threshold, seed = _checked(q, k, v, pos_key_layer, pos_query_layer, q.shape[1], sm_scale, position_buckets, max_relative_distance,
                                                dropout_p, seed, longest, longest, (seqlens_k,))
    if seqlens_k is not None:
        if seqlens_k.shape != q.shape[:1]:
            raise ValueError(f"seqlens_k must be [B={q.shape[0]}], got {tuple(seqlens_k.shape)}")
        seqlens_k = seqlens_k.to(torch.int32).contiguous()
    return _Attention.apply(q, k, v, pk, pq, seqlens_k, None, seed, longest, scale, int(position_buckets), int(max_relative_distance), threshold)


def trainable_attention_with_disentangled_varlen(q, k, v, pos_key_layer: Optional[torch.Tensor], pos_query_layer: Optional[torch.Tensor],
                                                 cu_seqlens: torch.Tensor, max_seqlen: int, sm_scale: Optional[float] = None,
                                                 position_buckets: int = 0, max_relative_distance: int = 0, *, dropout_p: float = 0.0,
                                                 seed: Optional[torch.Tensor] = None):
    """``trainable_attention_with_disentangled`` of packed sequences: q, k, v ``[total_tokens, H, D]``, cu_seqlens int32 ``[B+1]`` running sums of the lengths with a
    leading 0, max_seqlen the longest (an upper bound is fine; what it cuts off, and tokens of no sequence, are zeros in the result and in the
    gradients).  No host synchronisation."""
    o = _lib.host().train_attention(q, k, v, pos_key_layer, pos_query_layer, sm_scale, position_buckets, max_relative_distance, None, cu_seqlens, max_seqlen, dropout_p, seed)
    if o is not None:
        return o
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k, v must be [total_tokens, H, D]")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a 1-D tensor of B+1 offsets")
    longest = max(int(max_seqlen), 1)
    scale, (pk, pq), threshold, seed = _checked(q, k, v, pos_key_layer, pos_query_layer, q.shape[1], sm_scale, position_buckets, max_relative_distance,
                                                dropout_p, seed, longest, min(longest, q.shape[0]), (cu_seqlens,))
    return _Attention.apply(q, k, v, pk, pq, None, cu_seqlens.to(torch.int32).contiguous(), seed, longest, scale, int(position_buckets),
                            int(max_relative_distance), threshold)
