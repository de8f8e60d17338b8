"""Operators of an encoder's layers around the token block: attention.

With the token block's operators they make the token states that ``maxsim`` scores out of token
ids.  (Extension: the reference starts from finished embeddings.)  As in ``block``, each comes as
a verb that torch autograd records and as the forward and pullback it is made of:

    o = attention(q, k, v, qmask, kmask, ...)    softmax(scale q k^T) v over heads, one kernel

The heads of a token lie side by side: q is (B, T, heads, dim) or (T, heads, dim), k and v the
same with as many or fewer heads.  Any strides do, a head's values contiguous, so slices of one
projection's output need no copy.  All are of one feature type (float32, float16, bfloat16); sums
run in fp32 and outputs are rounded once.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import boundary
from .block import _cotangent
from .errors import ArgumentError, DimensionMismatch


# ---- attention -----------------------------------------------------------------------------

class AttentionKept(NamedTuple):
    """What ``attention_pullback`` needs of the forward beside its output: base-2 logarithms of the
    rows' sums, and what the output's rounding left (None in float32)."""
    lse: torch.Tensor
    rest: torch.Tensor | None


def _attention_options(q, k, v, qmask, kmask, cu_q, cu_k, max_q, max_k, causal, window, scale):
    """Shapes of the heads and the options as the boundary takes them (it checks the rest)."""
    if q.dim() not in (3, 4) or k.dim() != q.dim() or v.shape != k.shape:
        raise DimensionMismatch("attention takes q (B, Tq, heads, dim) and k, v (B, Tk, kv_heads, dim), "
                                "or all of them without B")
    if q.shape[-1] != k.shape[-1] or q.shape[:-3] != k.shape[:-3]:
        raise DimensionMismatch(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch or dim")
    if k.shape[-2] == 0 and q.shape[-2] > 0 or k.shape[-2] > 0 and q.shape[-2] % k.shape[-2]:
        raise DimensionMismatch(f"{q.shape[-2]} query heads cannot share {k.shape[-2]} key heads evenly")
    if (cu_q is None) != (cu_k is None):
        raise ArgumentError("ragged attention needs cu_q and cu_k (the same one for self-attention)")
    if cu_q is not None:
        if q.dim() != 3:
            raise DimensionMismatch("ragged attention takes token rows (tokens, heads, dim)")
        if qmask is not None or kmask is not None:
            raise ArgumentError("masks go with padded sequences, not with cu_q and cu_k")
        max_q = q.shape[0] if max_q is None else int(max_q)
        max_k = k.shape[0] if max_k is None else int(max_k)
        if max_q < 0 or max_k < 0:
            raise ArgumentError("max_q and max_k must be >= 0")
    elif max_q is not None or max_k is not None:
        raise ArgumentError("max_q and max_k go with cu_q and cu_k")
    if window is not None and window < 0:
        raise ArgumentError("window must be >= 0, or None")
    if scale is None:
        scale = max(q.shape[-1], 1) ** -0.5
    return (qmask, kmask, cu_q, cu_k, max_q or 0, max_k or 0, float(scale), 1 if causal else 0,
            -1 if window is None else int(window))


def attention_forward(q, k, v, qmask=None, kmask=None, *, cu_q=None, cu_k=None, max_q=None, max_k=None,
                      causal=False, window=None, scale=None, keep=False):
    """o (q's shape), dense; with ``keep`` (o, kept) for ``attention_pullback``.  See ``attention``."""
    options = _attention_options(q, k, v, qmask, kmask, cu_q, cu_k, max_q, max_k, causal, window, scale)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = rest = None
    if keep:
        *lead, tokens, heads, _ = q.shape
        shared = k.shape[-2]
        lse = torch.empty((*lead, shared, tokens * (heads // max(shared, 1))), dtype=torch.float32,
                          device=q.device)
        rest = None if q.dtype == torch.float32 else torch.empty_like(o)
    boundary.launch_attention(o, lse, rest, q, k, v, *options)
    return (o, AttentionKept(lse, rest)) if keep else o


def attention_pullback(do, q, k, v, o, kept, qmask=None, kmask=None, *, cu_q=None, cu_k=None, max_q=None,
                       max_k=None, causal=False, window=None, scale=None):
    """(dq, dk, dv), dense, for the cotangent do of o; o and kept are the forward's, the other
    arguments as they were there."""
    options = _attention_options(q, k, v, qmask, kmask, cu_q, cu_k, max_q, max_k, causal, window, scale)
    do = _cotangent(do, q.shape, q, "do")
    if do is None:
        raise DimensionMismatch("do: missing")
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    boundary.attention_apply_pullback(dq, dk, dv, do, o, kept.lse, kept.rest, q, k, v, *options)
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, qmask, kmask, cu_q, cu_k, args):
        o, kept = attention_forward(q, k, v, qmask, kmask, cu_q=cu_q, cu_k=cu_k, keep=True, **args)
        ctx.save_for_backward(q, k, v, o, *kept, qmask, kmask, cu_q, cu_k)
        ctx.args = args
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, rest, qmask, kmask, cu_q, cu_k = ctx.saved_tensors
        grads = attention_pullback(do, q, k, v, o, AttentionKept(lse, rest), qmask, kmask, cu_q=cu_q,
                                   cu_k=cu_k, **ctx.args)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 5


def attention(q, k, v, qmask=None, kmask=None, *, cu_q=None, cu_k=None, max_q=None, max_k=None,
              causal=False, window=None, scale=None):
    """softmax(scale q kᵀ) v over heads, recorded by autograd.

    q (B, Tq, heads, dim), k and v (B, Tk, kv_heads, dim), or all without B; query heads h * n ..
    h * n + n - 1 share key head h where there are n times as many.  scale is dim ** -0.5 unless
    given.  A query sees the keys that

    * its masks leave: qmask (B, Tq) and kmask (B, Tk), Bool.  A masked query gives zeros; what lies
      behind a mask, or its cotangent, is not read;
    * are not behind it (``causal``) and at most ``window`` tokens away, the last query beside the
      last key.

    A query that sees none gives zeros.  Ragged sequences come as token rows q (Nq, heads, dim), k and
    v (Nk, kv_heads, dim) with the 1-based Int32 ``cu`` of a ``PackedSeq`` (cu_q and cu_k, one array
    twice for self-attention) and the longest lengths, max_q and max_k (the token counts if not given:
    as right, and slower); masks are for padded sequences.

    The pullback computes the probabilities again; kept for it are the inputs, the output, and 4
    bytes a query and head and (16-bit types) what the output's rounding left.  dim is at most 128."""
    args = dict(max_q=max_q, max_k=max_k, causal=causal, window=window, scale=scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, qmask, kmask, cu_q, cu_k, args)
    return attention_forward(q, k, v, qmask, kmask, cu_q=cu_q, cu_k=cu_k, **args)
