"""Operators of a token block: gated feed-forward and the norms around it.

A token block makes the embeddings that ``maxsim`` scores out of an encoder's token
states.  (Extension: the reference starts from finished embeddings.)  Each operator comes
as a verb that torch autograd records (``gated_ffn``, ``block_norm``) and as the forward and
pullback it is made of (``*_forward``, ``*_pullback``), all on the HIP kernels of the library:

    h = gated_ffn(x, wg, wu, act)           act(x wg^T) * (x wu^T), one kernel
    r, n = block_norm(x, f, ...)            r = x + scale * gate * norm(f) * post_weight
                                            n = norm(r) * pre_weight, one kernel

Token states have the package's shapes ((T, dim) or (B, T, dim), any leading dimensions),
weights are (hidden, dim) and (dim,), all in one feature type (float32, float16, bfloat16).
Sums run in fp32 and each output is rounded once; what the pullbacks hold between their sums
has more bits than the feature type.  Arrays must be dense and on the device.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import boundary
from .errors import ArgumentError, DimensionMismatch

ACTIVATIONS = ("silu", "gelu", "gelu_tanh")
NORMS = ("rms", "layer")


def _code(value, names, what):
    try:
        return names.index(value)
    except ValueError:
        raise ArgumentError(f"{what} must be one of {', '.join(names)}, got {value!r}") from None


def _cotangent(d, shape, proto, what):
    """A cotangent as a dense array of the feature eltype (None: zero)."""
    if d is None:
        return None
    if not isinstance(d, torch.Tensor) or d.shape != shape:
        raise DimensionMismatch(f"{what} must have the shape {tuple(shape)}")
    if d.dtype != proto.dtype or d.device != proto.device:
        d = d.to(device=proto.device, dtype=proto.dtype)
    return d.contiguous()


# ---- gated feed-forward --------------------------------------------------------------------

def _hidden(x, wg, wu):
    """The weights' hidden units (the boundary checks shapes, eltypes and devices)."""
    if x.dim() < 1 or wg.dim() != 2 or wu.dim() != 2:
        raise DimensionMismatch("gated_ffn takes x (..., dim) and weights (hidden, dim)")
    return wg.shape[0]


def gated_ffn_forward(x, wg, wu, act="silu"):
    """h (..., hidden) = act(x wgᵀ) * (x wuᵀ) for x (..., dim), wg and wu (hidden, dim)."""
    code = _code(act, ACTIVATIONS, "act")
    h = x.new_empty((*x.shape[:-1], _hidden(x, wg, wu)))
    boundary.launch_gated_ffn(h, x, wg, wu, code)
    return h


def gated_ffn_pullback(dh, x, wg, wu, act="silu", need_dx=True, need_dw=True):
    """(dx, dwg, dwu) for the cotangent dh (..., hidden); None where not needed."""
    code = _code(act, ACTIVATIONS, "act")
    dh = _cotangent(dh, (*x.shape[:-1], _hidden(x, wg, wu)), x, "dh")
    if dh is None:
        raise DimensionMismatch("dh: missing")
    dx = torch.empty_like(x) if need_dx else None
    dwg, dwu = (torch.empty_like(wg), torch.empty_like(wu)) if need_dw else (None, None)
    boundary.gated_ffn_apply_pullback(dx, dwg, dwu, dh, x, wg, wu, code)
    return dx, dwg, dwu


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, act):
        ctx.save_for_backward(x, wg, wu)
        ctx.act = act
        return gated_ffn_forward(x, wg, wu, act)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        need = ctx.needs_input_grad
        x, wg, wu = ctx.saved_tensors
        dx, dwg, dwu = gated_ffn_pullback(dh, x, wg, wu, ctx.act, need[0], need[1] or need[2])
        return dx, dwg if need[1] else None, dwu if need[2] else None, None


def gated_ffn(x, wg, wu, act="silu"):
    """act(x wgᵀ) * (x wuᵀ), recorded by autograd.  act: "silu" (SwiGLU), "gelu" (the exact
    one) or "gelu_tanh".  Nothing but the inputs is kept for the pullback."""
    return _GatedFFN.apply(x, wg, wu, act)


# ---- norms around a block ------------------------------------------------------------------

def _norm_check(x, f, gate, post_weight, pre_weight):
    """How many neighbouring rows share a gate vector (the boundary checks shapes, eltypes and
    devices)."""
    if x.dim() < 1:
        raise DimensionMismatch("block_norm takes x (..., dim)")
    if f is None:
        if gate is not None or post_weight is not None:
            raise ArgumentError("gate and post_weight need the branch f")
        if pre_weight is None:
            raise ArgumentError("block_norm has nothing to compute without f and pre_weight")
    return _gate_rows(x, gate)


def _gate_rows(x, gate):
    if gate is None:
        return max(x.shape[:-1].numel(), 1)
    lead = gate.dim() - 1
    if lead < 0 or lead > x.dim() - 1 or gate.shape != x.shape[:lead] + x.shape[-1:]:
        raise DimensionMismatch(
            f"gate must be (dim,) or x's leading dimensions and dim: got {tuple(gate.shape)} for "
            f"x {tuple(x.shape)}")
    return max(x.shape[lead:-1].numel(), 1)


def block_norm_forward(x, f=None, *, gate=None, post_weight=None, pre_weight=None, scale=1.0,
                       kind="rms", eps=1e-6):
    """(r, n): r = x + scale * gate * z with z = norm(f) * post_weight (f itself without
    post_weight), n = norm(r) * pre_weight.  Without f, r is x; without pre_weight, n is None."""
    code = _code(kind, NORMS, "kind")
    gate_rows = _norm_check(x, f, gate, post_weight, pre_weight)
    r = None if f is None else torch.empty_like(x)
    n = None if pre_weight is None else torch.empty_like(x)
    boundary.launch_block_norm(r, n, x, f, gate, post_weight, pre_weight, code, scale, eps, gate_rows)
    return (x if f is None else r), n


def block_norm_pullback(dr, dn, x, f=None, *, gate=None, post_weight=None, pre_weight=None,
                        scale=1.0, kind="rms", eps=1e-6):
    """(dx, df, dgate, dpost_weight, dpre_weight) for the cotangents of r and n (either may be
    None: zero); None for an input that was not given."""
    code = _code(kind, NORMS, "kind")
    gate_rows = _norm_check(x, f, gate, post_weight, pre_weight)
    dr, dn = _cotangent(dr, x.shape, x, "dr"), _cotangent(dn, x.shape, x, "dn")
    if dn is not None and pre_weight is None:
        raise ArgumentError("dn needs pre_weight")
    grads = [None if t is None else torch.empty_like(t) for t in (x, f, gate, post_weight, pre_weight)]
    if gate is not None and x.numel() == 0:
        grads[2].zero_()  # a gate of no rows
    boundary.block_norm_apply_pullback(*grads, dr, dn, x, f, gate, post_weight, pre_weight, code,
                                       scale, eps, gate_rows)
    return tuple(grads)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, post_weight, pre_weight, scale, kind, eps):
        ctx.save_for_backward(x, f, gate, post_weight, pre_weight)
        ctx.args = dict(scale=scale, kind=kind, eps=eps)
        r, n = block_norm_forward(x, f, gate=gate, post_weight=post_weight, pre_weight=pre_weight,
                                  **ctx.args)
        ctx.set_materialize_grads(False)
        return (None if f is None else r), n

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, dn):
        x, f, gate, post_weight, pre_weight = ctx.saved_tensors
        grads = block_norm_pullback(dr, dn, x, f, gate=gate, post_weight=post_weight,
                                    pre_weight=pre_weight, **ctx.args)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 3


def block_norm(x, f=None, *, gate=None, post_weight=None, pre_weight=None, scale=1.0, kind="rms",
               eps=1e-6):
    """(r, n) as ``block_norm_forward``, recorded by autograd: the end of one block (norm of its
    branch f, gate, residual) and the start of the next (norm of the sum) in one pass.

    kind: "rms" or "layer"; gate: (dim,), or one vector for each of x's leading indices -- (B,
    dim) for x (B, T, dim) gates each sequence, x's own shape each token.  For the first norm
    of a model leave out f, for the last residual leave out pre_weight."""
    r, n = _BlockNorm.apply(x, f, gate, post_weight, pre_weight, float(scale), kind, float(eps))
    return (x if f is None else r), n
