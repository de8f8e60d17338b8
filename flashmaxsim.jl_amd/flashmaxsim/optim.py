"""AdamW over many tensors at once, with its moments in 32 or in 8 bits.

The step that uses MaxSim's gradients (extension; the reference leaves the optimiser to its
caller).  All tensors of a step go through one kernel, up to 480 a launch, in place:

    m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

in fp32.  With fp32 masters beside 16-bit parameters the step works on the masters and the
parameters become their roundings.

8-bit moments (``Moment8``) hold a code for each element and an fp32 scale for every 256
neighbouring elements, the largest magnitude among them: m as int8 codes with the value
sign(c) (c/127)^2 scale, v as uint8 codes with the value (c/255)^4 scale.
"""
from __future__ import annotations

import numpy as np
import torch

from . import boundary
from .errors import ArgumentError, DimensionMismatch

MOMENT_BLOCK = 256
# Entries of the library's tables (fms_adamw_tensor, fms_moment8).
_ADAMW_ENTRY = np.dtype([(k, "u8") for k in ("p", "m", "v", "master", "m_scale", "v_scale")]
                        + [("n", "i8"), ("p_dtype", "i8")])
_numel, _address, _dtype = torch.Tensor.numel, torch.Tensor.data_ptr, torch.Tensor.dtype.__get__
_MOMENT_ENTRY = np.dtype([("codes", "u8"), ("scales", "u8"), ("values", "u8"), ("n", "i8"),
                          ("is_signed", "i8")])


class Moment8:
    """A moment in 8 bits: ``codes`` (int8 for m, uint8 for v) in the parameter's shape and
    ``scales``, one float32 for each 256 of its elements in memory order."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype not in (torch.int8, torch.uint8):
            raise ArgumentError(f"moment codes are int8 or uint8, got {codes.dtype}")
        if scales.dtype != torch.float32:
            raise ArgumentError(f"moment scales are float32, got {scales.dtype}")
        if scales.numel() != -(-codes.numel() // MOMENT_BLOCK):
            raise DimensionMismatch(f"{scales.numel()} moment scales for {codes.numel()} codes")
        self.codes, self.scales = codes, scales

    @classmethod
    def zeros(cls, p: torch.Tensor, signed: bool) -> "Moment8":
        """The moment of a first step: m (signed) or v of the parameter p."""
        return cls(torch.zeros(p.shape, dtype=torch.int8 if signed else torch.uint8, device=p.device),
                   torch.zeros(-(-p.numel() // MOMENT_BLOCK), dtype=torch.float32, device=p.device))

    def __repr__(self):
        return f"Moment8(codes={tuple(self.codes.shape)} {self.codes.dtype})"


def moment_values(moments, out=None):
    """The float32 values of Moment8s, many at once; ``out``: tensors to write them to."""
    moments = list(moments)
    if out is None:
        out = [torch.empty(m.codes.shape, dtype=torch.float32, device=m.codes.device)
               for m in moments]
    out = list(out)
    if len(out) != len(moments):
        raise DimensionMismatch(f"{len(out)} outputs for {len(moments)} moments")
    if not moments:
        return out
    codes, scales = [m.codes for m in moments], [m.scales for m in moments]
    dev = boundary.require_device_many(codes, scales, out)
    numels = [c.numel() for c in codes]
    if any(o.dtype != torch.float32 for o in out):
        raise ArgumentError("moment values are float32")
    if [o.numel() for o in out] != numels:
        raise DimensionMismatch("as many values as codes")
    table = np.empty(len(moments), _MOMENT_ENTRY)
    for name, ts in (("codes", codes), ("scales", scales), ("values", out)):
        table[name] = [t.data_ptr() for t in ts]
    table["n"] = numels
    table["is_signed"] = [c.dtype == torch.int8 for c in codes]
    boundary.moment_values(table, dev)
    return out


class AdamW:
    """AdamW over a list of parameters.

    bits: 32 (float32 moments) or 8 (``Moment8``); masters: True to keep float32 copies of
    16-bit parameters, or a list of them (None where a parameter has none); moments: a pair
    of lists (m, v) to go on from, with ``step`` the steps already taken.

    A step's number, rate and addresses are arguments of its kernels: captured in a graph it
    would repeat the same step."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, bits=32,
                 masters=None, moments=None, step=0):
        self.params = list(params)
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.steps = int(step)
        if bits not in (8, 32):
            raise ArgumentError(f"moments are held in 32 or in 8 bits, got {bits!r}")
        b1, b2 = self.betas
        if not (0 <= b1 < 1 and 0 <= b2 < 1 and eps >= 0 and self.steps >= 0):
            raise ArgumentError(f"AdamW: betas {self.betas}, eps {eps}, step {step}")
        self._device = boundary.require_device(*self.params)
        if len(set(map(id, self.params))) != len(self.params):
            raise ArgumentError("AdamW: a parameter is given twice")
        codes = [boundary.dtype_code(p) for p in self.params]
        if moments is None:
            if bits == 8:
                moments = ([Moment8.zeros(p, True) for p in self.params],
                           [Moment8.zeros(p, False) for p in self.params])
            else:
                moments = tuple([torch.zeros_like(p, dtype=torch.float32) for p in self.params]
                                for _ in range(2))
        self.m, self.v = tuple(moments[0]), tuple(moments[1])
        if masters is True:
            masters = [None if p.dtype == torch.float32 else p.detach().float() for p in self.params]
        self.masters = (None,) * len(self.params) if not masters else tuple(masters)
        if not len(self.params) == len(self.m) == len(self.v) == len(self.masters):
            raise DimensionMismatch("AdamW: as many moments and masters as parameters")
        # the table of the library, and what its addresses belong to
        self._numels, self._dtypes = [p.numel() for p in self.params], [p.dtype for p in self.params]
        self._held = []
        self._table = np.zeros(len(self.params), _ADAMW_ENTRY)
        self._table["n"], self._table["p_dtype"] = self._numels, codes
        for e, p, m, v, w in zip(self._table, self.params, self.m, self.v, self.masters):
            self._place(e, p, m, v, w)
        self._place_params()

    def _place_params(self):
        """Checks the parameters and notes where they lie.  Their memory is held until they are
        seen elsewhere, so it is theirs as long as they are seen there."""
        if ([p.numel() for p in self.params] != self._numels
                or [p.dtype for p in self.params] != self._dtypes):
            raise DimensionMismatch("AdamW: a parameter has changed its size or eltype")
        if self.params and boundary.require_device(*self.params) != self._device:
            raise ArgumentError("FlashMaxSim requires colocated arrays (same device)")
        memory = [p.detach() for p in self.params]
        addresses = list(map(_address, memory))
        self._table["p"] = addresses
        self._check_apart()
        plan = boundary.adamw_plan(self._table)
        if self.params:
            self._device_plan = torch.from_numpy(plan).to(self._device)
            self._plan_stream = boundary.stream_handle(self._device)
        self._memory, self._addresses, self._plan = memory, addresses, plan  # (all checked)

    def _check_apart(self):
        """A step writes every array from workgroups in no order: none may share memory."""
        t, scales = self._table, -(-self._table["n"] // MOMENT_BLOCK) * 4
        moment = np.where(t["m_scale"] != 0, 1, 4) * t["n"]
        sizes = np.concatenate([t["n"] * [p.element_size() for p in self.params], moment, moment,
                                t["n"] * 4, scales, scales])
        starts = np.concatenate([t[k] for k in ("p", "m", "v", "master", "m_scale", "v_scale")])
        given = (starts != 0) & (sizes > 0)
        starts, sizes = starts[given].astype(np.int64), sizes[given].astype(np.int64)
        order = np.argsort(starts)
        starts, ends = starts[order], (starts + sizes)[order]
        if (starts[1:] < ends[:-1]).any():
            raise ArgumentError("AdamW: parameters, moments and masters must not share memory")

    def _place(self, e, p, m, v, master):
        if isinstance(m, Moment8) != isinstance(v, Moment8):
            raise ArgumentError("AdamW: both moments of a parameter in 32 or both in 8 bits")
        if isinstance(m, Moment8):
            boundary.require_device(p, m.codes, m.scales, v.codes, v.scales)
            if m.codes.dtype != torch.int8 or v.codes.dtype != torch.uint8:
                raise ArgumentError("AdamW: m has int8 codes and v uint8 codes")
            e["m_scale"], e["v_scale"] = m.scales.data_ptr(), v.scales.data_ptr()
            self._held += [m.scales, v.scales]
            m, v = m.codes, v.codes
        else:
            boundary.require_device(p, m, v)
            if m.dtype != torch.float32 or v.dtype != torch.float32:
                raise ArgumentError("AdamW: moments are float32 or Moment8")
        if not m.numel() == v.numel() == p.numel():
            raise DimensionMismatch("AdamW: the moments have their parameter's size")
        e["m"], e["v"] = m.data_ptr(), v.data_ptr()
        self._held += [m, v, master]
        if master is not None:
            boundary.require_device(p, master)
            if master.dtype != torch.float32:
                raise ArgumentError("AdamW: masters are float32")
            if master.numel() != p.numel():
                raise DimensionMismatch("AdamW: a master has its parameter's size")
            e["master"] = master.data_ptr()

    def step(self, grads=None, lr=None, grad_scale=1.0):
        """One step, in place.  grads: one per parameter, None to leave it as it is (default: the
        parameters' .grad); lr: instead of the optimiser's; grad_scale: multiplies the
        gradients (loss scaling, clipping)."""
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise DimensionMismatch(f"{len(grads)} gradients for {len(self.params)} parameters")
        params, numels = self.params, self._numels
        if (list(map(_address, params)) != self._addresses or list(map(_numel, params)) != numels
                or not all(map(torch.Tensor.is_contiguous, params))):
            self._place_params()
        addresses = np.zeros(len(params), np.uint64)
        keep = slice(None)
        if [g for g in grads if g is None]:
            keep = [i for i, g in enumerate(grads) if g is not None]
            params, grads = [params[i] for i in keep], [grads[i] for i in keep]
            numels = [numels[i] for i in keep]
        if not grads:
            return
        if boundary.require_device_many(grads) != self._device:
            raise ArgumentError("FlashMaxSim requires colocated arrays (same device)")
        if list(map(_numel, grads)) != numels:
            raise DimensionMismatch("AdamW: a gradient has its parameter's size")
        addresses[keep] = list(map(_address, grads))
        dtypes = np.zeros(len(addresses), np.int32)
        one_type = len(set(map(_dtype, grads))) == 1
        dtypes[keep] = (boundary.dtype_code(grads[0]) if one_type
                        else [boundary.dtype_code(g) for g in grads])
        if boundary.stream_handle(self._device) != self._plan_stream:
            # (its memory goes back to the stream it came from, past steps on this one)
            self._device_plan.record_stream(torch.cuda.current_stream(self._device))
        boundary.adamw_step(self._plan, self._device_plan, addresses, dtypes, self.steps + 1,
                            self.lr if lr is None else lr, self.betas, self.eps, self.weight_decay,
                            grad_scale, self._device)
        self.steps += 1
        torch.autograd.graph.increment_version(params)

    def moment_values(self, out=None):
        """(m, v) as float32 lists; out: such a pair to write the values of 8-bit moments to."""
        both = self.m + self.v
        to = [None] * len(both) if out is None else list(out[0]) + list(out[1])
        at = [i for i, m in enumerate(both) if isinstance(m, Moment8)]
        got = moment_values([both[i] for i in at], None if out is None else [to[i] for i in at])
        values = list(both)
        for i, t in zip(at, got):
            values[i] = t
        return values[:len(self.m)], values[len(self.m):]

    def __repr__(self):
        bits = "8" if self.m and isinstance(self.m[0], Moment8) else "32"
        return f"AdamW({len(self.params)} tensors, {bits}-bit moments, step {self.steps})"
