"""Operators of an encoder's layers around the token block: token lookup, the norm and rotation of
queries and keys, attention.

With the token block's operators they make the token states that ``maxsim`` scores out of token
ids.  (Extension: the reference starts from finished embeddings.)  As in ``block``, each comes as
a verb that torch autograd records and as the forward and pullback it is made of:

    e = embed_tokens(ids, weight, scale)         rows of the table, scaled
    q, k = head_rotary(q, k, table, ...)         norm of each head, and its rotation by position
    o = attention(q, k, v, qmask, kmask, ...)    softmax(scale q k^T) v over heads, one kernel

The heads of a token lie side by side: q is (B, T, heads, dim) or (T, heads, dim), k and v the
same with as many or fewer heads.  Any strides do, a head's values contiguous, so slices of one
projection's output need no copy.  All are of one feature type (float32, float16, bfloat16); sums
run in fp32 and outputs are rounded once.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import boundary
from .block import NORMS, _code, _cotangent
from .errors import ArgumentError, DimensionMismatch

PAIRINGS = ("halves", "neighbours")


# ---- token lookup --------------------------------------------------------------------------

def embed_tokens_forward(ids, weight, scale=1.0):
    """e (*ids.shape, dim) = scale * weight[ids - 1]; see ``embed_tokens``."""
    if weight.dim() != 2:
        raise DimensionMismatch("embed_tokens takes a table (vocabulary, dim)")
    e = weight.new_empty((*ids.shape, weight.shape[1]))
    boundary.launch_embed_tokens(e, ids, weight, float(scale))
    return e


def embed_tokens_pullback(de, ids, vocabulary, scale=1.0):
    """dweight (vocabulary, dim) for the cotangent de (*ids.shape, dim): every row written."""
    if de.dim() != ids.dim() + 1 or vocabulary < 0:
        raise DimensionMismatch(f"de must be ids' shape and dim: got {tuple(de.shape)} for {tuple(ids.shape)}")
    dweight = de.new_empty((vocabulary, de.shape[-1]))
    boundary.embed_tokens_apply_pullback(dweight, de.contiguous(), ids, float(scale))
    return dweight


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.args = weight.shape[0], scale
        return embed_tokens_forward(ids, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, de):
        return None, embed_tokens_pullback(de, ctx.saved_tensors[0], *ctx.args), None


def embed_tokens(ids, weight, scale=1.0):
    """scale * weight[ids - 1], recorded by autograd: ids (Int32 or Int64, any shape) are 1-based rows of
    weight (vocabulary, dim), as every index of the package.  An id outside 1 .. vocabulary gives
    zeros and takes no part in the gradient; 0 pads.  The gradient is the whole table's, its sums in
    fp32 and in an order that the tokens' own fixes (partial sums, joined, for frequent ids)."""
    return _EmbedTokens.apply(ids, weight, scale)


# ---- norm and rotation of heads --------------------------------------------------------------

def rotary_table(positions, turned, base=10000.0, device=None):
    """(positions, turned) float32 for ``head_rotary``: row p, counted from 0, has the cosines and then the
    sines of p * base ** (-2 i / turned), i < turned / 2.  The angles are computed in 64 bits, in
    32 far positions would be off by much of a turn."""
    if positions < 0 or turned < 0 or turned % 2:
        raise ArgumentError("rotary_table takes counts >= 0, turned even")
    i = torch.arange(turned // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 / max(turned, 1) * i)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _rotary_codes(q, k, kind, pairing):
    qs = q.shape
    if len(qs) not in (3, 4):
        raise DimensionMismatch("head_rotary takes q (B, T, heads, dim) or (T, heads, dim)")
    if qs[-1] % 2:
        raise DimensionMismatch(f"head_rotary takes heads of an even number of values, got {qs[-1]}")
    return _code(kind, NORMS, "kind"), _code(pairing, PAIRINGS, "pairing")


def _dense_like(t):
    return None if t is None else t.new_empty(t.shape)


def head_rotary_forward(q, k, table, positions=None, *, q_weight=None, k_weight=None, kind="rms",
                        pairing="halves", eps=1e-6):
    """(q, k) with each head normed and rotated, dense; see ``head_rotary``."""
    codes = _rotary_codes(q, k, kind, pairing)
    out = _dense_like(q), _dense_like(k)
    boundary.launch_head_rotary(*out, q, k, table, positions, q_weight, k_weight, *codes, float(eps))
    return out


def head_rotary_pullback(dq_out, dk_out, q, k, table, positions=None, *, q_weight=None, k_weight=None,
                         kind="rms", pairing="halves", eps=1e-6):
    """(dq, dk, dq_weight, dk_weight) for the cotangents of both outputs (None: zero); None for what was not
    given."""
    codes = _rotary_codes(q, k, kind, pairing)
    cotangents = []
    for d, like, what in ((dq_out, q, "dq_out"), (dk_out, k, "dk_out")):
        d = None if like is None else _cotangent(d, like.shape, like, what)
        if d is None and like is not None:
            d = torch.zeros(like.shape, dtype=like.dtype, device=like.device)
        cotangents.append(d)
    grads = [_dense_like(t) for t in (q, k, q_weight, k_weight)]
    boundary.head_rotary_apply_pullback(*grads, *cotangents, q, k, table, positions, q_weight, k_weight,
                                        *codes, float(eps))
    return tuple(grads)


class _HeadRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, positions, args):
        ctx.save_for_backward(q, k, q_weight, k_weight, table, positions)
        ctx.args = args
        ctx.set_materialize_grads(False)
        return head_rotary_forward(q, k, table, positions, q_weight=q_weight, k_weight=k_weight, **args)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, q_weight, k_weight, table, positions = ctx.saved_tensors
        grads = head_rotary_pullback(dq, dk, q, k, table, positions, q_weight=q_weight, k_weight=k_weight,
                                     **ctx.args)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 3


def head_rotary(q, k, table, positions=None, *, q_weight=None, k_weight=None, kind="rms", pairing="halves",
                eps=1e-6):
    """(q, k) with each head normed and then rotated by its token's position, recorded by autograd.

    q (B, T, heads, dim), k (B, T, kv_heads, dim) or None, or both without B.  A head is normed over its
    values (kind "rms" or "layer") and multiplied by its weight (dim,); without a weight it is only
    rotated.  table (P, turned), as ``rotary_table`` makes it, has the cosines and sines of the first
    ``turned`` values of a head, taken in pairs (i, i + turned / 2) ("halves") or (2 i, 2 i + 1)
    ("neighbours"); the other values are not rotated.  positions, (T,) or (B, T), Int32 or Int64, are
    1-based rows of the table, token t takes row t without them.  A position that is none of the
    table's (0, say, for padding) gives zeros and takes no part in the gradients.  dim is even and
    at most 512."""
    args = dict(kind=kind, pairing=pairing, eps=eps)
    return _HeadRotary.apply(q, k, q_weight, k_weight, table, positions, args)


# ---- attention -----------------------------------------------------------------------------

class AttentionKept(NamedTuple):
    """What ``attention_pullback`` needs of the forward beside its output: the rows' largest q k (of the
    other sign under a negative scale; -inf where a query sees no key), and what the output's rounding
    left (None in float32)."""
    top: torch.Tensor
    rest: torch.Tensor | None


_MOST = 1 << 40  # more than any length or window: what passes 64 bits would lose its upper ones on the way


def _attention_options(q, k, v, qmask, kmask, cu_q, cu_k, max_q, max_k, causal, window, scale):
    """Shapes of the heads and the options as the boundary takes them (it checks the rest)."""
    qs, ks = q.shape, k.shape
    n = len(qs)
    if n not in (3, 4) or len(ks) != n:
        raise DimensionMismatch("attention takes q (B, Tq, heads, dim) and k, v (B, Tk, kv_heads, dim), "
                                "or all of them without B")
    if qs[-2] != ks[-2] and (not ks[-2] or not qs[-2] or qs[-2] % ks[-2]):
        raise DimensionMismatch(f"{qs[-2]} query heads cannot share {ks[-2]} key heads evenly")
    if cu_q is None and cu_k is None:
        if max_q is not None or max_k is not None:
            raise ArgumentError("max_q and max_k go with cu_q and cu_k")
        max_q = max_k = 0
    else:
        if cu_q is None or cu_k is None:
            raise ArgumentError("ragged attention needs cu_q and cu_k (the same one for self-attention)")
        if n != 3:
            raise DimensionMismatch("ragged attention takes token rows (tokens, heads, dim)")
        if qmask is not None or kmask is not None:
            raise ArgumentError("masks go with padded sequences, not with cu_q and cu_k")
        max_q = qs[0] if max_q is None else min(int(max_q), _MOST)
        max_k = ks[0] if max_k is None else min(int(max_k), _MOST)
        if max_q < 0 or max_k < 0:
            raise ArgumentError("max_q and max_k must be >= 0")
    if window is None:
        window = -1
    elif window < 0:
        raise ArgumentError("window must be >= 0, or None")
    if scale is None:
        scale = qs[-1] ** -0.5 if qs[-1] else 1.0
    return qmask, kmask, cu_q, cu_k, max_q, max_k, float(scale), 1 if causal else 0, min(int(window), _MOST)


def attention_forward(q, k, v, qmask=None, kmask=None, *, cu_q=None, cu_k=None, max_q=None, max_k=None,
                      causal=False, window=None, scale=None, keep=False):
    """o (q's shape), dense; with ``keep`` (o, kept) for ``attention_pullback``.  See ``attention``."""
    options = _attention_options(q, k, v, qmask, kmask, cu_q, cu_k, max_q, max_k, causal, window, scale)
    o = q.new_empty(q.shape)
    top = rest = None
    if keep:
        *lead, tokens, heads, _ = q.shape
        shared = k.shape[-2]
        top = torch.empty((*lead, shared, tokens * (heads // max(shared, 1))), dtype=torch.float32,
                          device=q.device)
        rest = None if q.dtype is torch.float32 else q.new_empty(q.shape)
    boundary.launch_attention(o, top, rest, q, k, v, *options)
    return (o, AttentionKept(top, rest)) if keep else o


def attention_pullback(do, q, k, v, o, kept, qmask=None, kmask=None, *, cu_q=None, cu_k=None, max_q=None,
                       max_k=None, causal=False, window=None, scale=None):
    """(dq, dk, dv), dense, for the cotangent do of o; o and kept are the forward's, the other
    arguments as they were there."""
    options = _attention_options(q, k, v, qmask, kmask, cu_q, cu_k, max_q, max_k, causal, window, scale)
    do = _cotangent(do, q.shape, q, "do")
    if do is None:
        raise DimensionMismatch("do: missing")
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    boundary.attention_apply_pullback(dq, dk, dv, do, o, kept.top, kept.rest, q, k, v, *options)
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
        q, k, v, o, top, rest, qmask, kmask, cu_q, cu_k = ctx.saved_tensors
        grads = attention_pullback(do, q, k, v, o, AttentionKept(top, rest), qmask, kmask, cu_q=cu_q,
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

    A query that sees none gives zeros.  What counts for some query should be finite: with ``causal`` or a
    window, a value that is not also makes results and gradients NaN of tokens close by that do not
    see it (those in reach of the same 64 keys or query rows).  Ragged sequences come as token rows q (Nq, heads, dim), k and
    v (Nk, kv_heads, dim) with the 1-based Int32 ``cu`` of a ``PackedSeq`` (cu_q and cu_k, one array
    twice for self-attention) and the longest lengths, max_q and max_k (the token counts if not given:
    as right, but the work is laid out for sequences of that length, so many of them take long, and very
    many are refused); masks are for padded sequences.

    The pullback computes the probabilities again; kept for it are the inputs, the output, and 4
    bytes a query and head and (16-bit types) what the output's rounding left.  dim is at most 128."""
    args = dict(max_q=max_q, max_k=max_k, causal=causal, window=window, scale=scale)
    # (forward mode's dual tensors need no gradient; the recorded call refuses them, as the other verbs do)
    if (forward_ad._current_level >= 0
            or torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return _Attention.apply(q, k, v, qmask, kmask, cu_q, cu_k, args)
    return attention_forward(q, k, v, qmask, kmask, cu_q=cu_q, cu_k=cu_k, **args)
