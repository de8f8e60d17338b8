"""AdamW over many tensors at once, with its moments in 32 or in 8 bits.

The step that uses MaxSim's gradients (extension; the reference leaves the optimiser to its
caller).  All tensors of a step go through one kernel, up to 480 a launch, in place:

    m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

with t the steps that the tensor itself has taken (those with a gradient for it), in fp32.  With fp32 masters beside 16-bit parameters the step works on the masters and the
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
_contiguous = torch.Tensor.is_contiguous
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


def _held(moment):
    """A moment's memory under a handle that no one else has."""
    if isinstance(moment, Moment8):
        return Moment8(moment.codes.detach(), moment.scales.detach())
    return moment.detach() if isinstance(moment, torch.Tensor) else moment


class AdamW:
    """AdamW over a list of parameters.

    bits: 32 (float32 moments) or 8 (``Moment8``); masters: True to keep float32 copies of
    16-bit parameters, or a list of them (None where a parameter has none); moments: a pair
    of lists (m, v) to go on from, with ``step`` the steps already taken, or the list of each
    parameter's own (``tensor_steps``): a step without a gradient for it is none of its.

    ``m``, ``v`` and ``masters`` are what the steps work on: for given ones, the memory that they
    were given in, held from then on.  To restore them, copy into them.  A parameter, or one of
    these, that is given other memory (``.data``, a Moment8's arrays) is stepped there.

    A step's number, rate and addresses are arguments of its kernels: captured in a graph it
    would repeat the same step."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, bits=32,
                 masters=None, moments=None, step=0):
        self.params = list(params)
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        if bits not in (8, 32):
            raise ArgumentError(f"moments are held in 32 or in 8 bits, got {bits!r}")
        if np.ndim(step) and len(step) != len(self.params):
            raise DimensionMismatch(f"{len(step)} numbers of steps for {len(self.params)} parameters")
        self._tensor_steps = np.zeros(len(self.params), np.int64)
        self._tensor_steps[:] = step
        self._steps = int(np.max(step, initial=0))
        b1, b2 = self.betas
        if not (0 <= b1 < 1 and 0 <= b2 < 1 and eps >= 0 and np.min(step, initial=0) >= 0):
            raise ArgumentError(f"AdamW: betas {self.betas}, eps {eps}, step {step}")
        self._device = boundary.require_device(*self.params)
        if len(set(map(id, self.params))) != len(self.params):
            raise ArgumentError("AdamW: a parameter is given twice")
        codes = [boundary.dtype_code(p) for p in self.params]
        if moments is not None:
            moments = [map(_held, ms) for ms in moments]
        elif bits == 8:
            moments = ([Moment8.zeros(p, signed) for p in self.params] for signed in (True, False))
        else:
            moments = ([torch.zeros_like(p, dtype=torch.float32) for p in self.params] for _ in range(2))
        self._m, self._v = map(tuple, moments)
        if masters is True:
            masters = [None if p.dtype == torch.float32 else p.detach().float() for p in self.params]
        elif masters:
            masters = map(_held, masters)
        self._masters = tuple(masters) if masters else (None,) * len(self.params)
        if not len(self.params) == len(self._m) == len(self._v) == len(self._masters):
            raise DimensionMismatch("AdamW: as many moments and masters as parameters")
        # Handles of the moments' and masters' memory once anyone else has seen them, and so can
        # have moved them: None until then.
        self._state_memory = None
        # the table of the library
        self._numels, self._dtypes = [p.numel() for p in self.params], [p.dtype for p in self.params]
        self._table = np.zeros(len(self.params), _ADAMW_ENTRY)
        self._table["n"], self._table["p_dtype"] = self._numels, codes
        self._home = boundary.stream_handle(self._device) if self.params else None
        self._place()

    @property
    def steps(self):
        """The steps taken; set, those of every tensor."""
        return self._steps

    @steps.setter
    def steps(self, n):
        self._steps = int(n)
        self._tensor_steps[:] = self._steps

    @property
    def tensor_steps(self):
        """The steps that each tensor has taken."""
        return self._tensor_steps.tolist()

    @property
    def m(self):
        self._show()
        return self._m

    @property
    def v(self):
        self._show()
        return self._v

    @property
    def masters(self):
        self._show()
        return self._masters

    def _show(self):
        if self._state_memory is None:
            self._state_memory = [t.detach() for t in self._arrays()]

    def _state(self):
        """The moments, masters and scales by their names in the library's table, None where a
        parameter has none."""
        m, v = self._m, self._v
        eight = [isinstance(a, Moment8) for a in m]
        if eight != [isinstance(a, Moment8) for a in v]:
            raise ArgumentError("AdamW: both moments of a parameter in 32 or both in 8 bits")
        if not any(eight):
            none = (None,) * len(m)
            return {"m": m, "v": v, "master": self._masters, "m_scale": none, "v_scale": none}
        return {"m": [a.codes if e else a for a, e in zip(m, eight)],
                "v": [a.codes if e else a for a, e in zip(v, eight)], "master": self._masters,
                "m_scale": [a.scales if e else None for a, e in zip(m, eight)],
                "v_scale": [a.scales if e else None for a, e in zip(v, eight)]}

    def _arrays(self):
        return [t for ts in self._state().values() for t in ts if t is not None]

    def _check_state(self, state):
        """Types and sizes of what _state gives."""
        blocks = [-(-n // MOMENT_BLOCK) for n in self._numels]
        eight = [s is not None for s in state["m_scale"]]
        for name, ts in state.items():
            code = {"m": torch.int8, "v": torch.uint8}.get(name)
            for t, n, b, e in zip(ts, self._numels, blocks, eight):
                if t is None:
                    continue
                if t.dtype != (code if code and e else torch.float32):
                    raise ArgumentError("AdamW: moments are float32, or Moment8 with int8 codes for m and uint8 "
                                        "codes for v; masters are float32")
                if t.numel() != (b if name.endswith("scale") else n):
                    raise DimensionMismatch("AdamW: moments and masters have their parameter's size")

    def _place(self):
        """Checks every array of a step and notes where it lies, in the library's plan.  The
        memory of what can be moved is held until it is seen elsewhere, so it is the array's own
        as long as that is seen there."""
        params = self.params
        if list(map(_numel, params)) != self._numels or list(map(_dtype, params)) != self._dtypes:
            raise DimensionMismatch("AdamW: a parameter has changed its size or eltype")
        state = self._state()
        arrays = [t for ts in state.values() for t in ts if t is not None]
        if params and boundary.require_device_many(params, arrays) != self._device:
            raise ArgumentError("FlashMaxSim requires colocated arrays (same device)")
        self._check_state(state)
        memory = [p.detach() for p in params]
        addresses = list(map(_address, memory))
        self._table["p"] = addresses
        for name, ts in state.items():
            self._table[name] = [0 if t is None else t.data_ptr() for t in ts]
        self._check_apart()
        plan = boundary.adamw_plan(self._table)
        if params:
            self._device_plan = torch.from_numpy(plan).to(self._device)
            # streams that the memory of what the optimiser has made is safe on
            self._streams = {boundary.stream_handle(self._device)} & {self._home}
        self._memory, self._addresses, self._plan = memory, addresses, plan  # (all checked)
        self._state_at = list(map(_address, arrays))
        if self._state_memory is not None:
            self._state_memory = [t.detach() for t in arrays]

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

    def _moved(self):
        """Whether an array does not lie where the plan has it."""
        params = self.params
        if (list(map(_address, params)) != self._addresses or list(map(_numel, params)) != self._numels
                or not all(map(_contiguous, params))):
            return True
        # (where they lie is enough: that memory is held.  444 of them take 34 us of host time beside
        # a step's 64)
        return self._state_memory is not None and list(map(_address, self._arrays())) != self._state_at

    def step(self, grads=None, lr=None, grad_scale=1.0):
        """One step, in place.  grads: one per parameter, None to leave it as it is (default: the
        parameters' .grad); lr: instead of the optimiser's; grad_scale: multiplies the
        gradients (loss scaling, clipping).  Gradients are only read; they must not lie in the
        memory of parameters, moments or masters."""
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise DimensionMismatch(f"{len(grads)} gradients for {len(self.params)} parameters")
        params, numels = self.params, self._numels
        if self._moved():
            self._place()
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
        stream = boundary.stream_handle(self._device)
        if stream not in self._streams:
            # (memory goes back to the stream it came from, past steps on this one)
            current = torch.cuda.current_stream(self._device)
            for t in self._arrays() + [self._device_plan]:
                t.record_stream(current)
            self._streams.add(stream)
        boundary.adamw_step(self._plan, self._device_plan, addresses, dtypes, self._tensor_steps + 1,
                            self.lr if lr is None else lr, self.betas, self.eps, self.weight_decay,
                            grad_scale, self._device)
        self._steps += 1
        self._tensor_steps[keep] += 1
        torch.autograd.graph.increment_version(params)

    def moment_values(self, out=None):
        """(m, v) as float32 lists; out: such a pair to write the values of 8-bit moments to."""
        both = self._m + self._v
        if not all(isinstance(m, Moment8) for m in both):
            self._show()
        to = [None] * len(both) if out is None else list(out[0]) + list(out[1])
        at = [i for i, m in enumerate(both) if isinstance(m, Moment8)]
        got = moment_values([both[i] for i in at], None if out is None else [to[i] for i in at])
        values = list(both)
        for i, t in zip(at, got):
            values[i] = t
        return values[:len(self._m)], values[len(self._m):]

    def __repr__(self):
        bits = "8" if self._m and isinstance(self._m[0], Moment8) else "32"
        return f"AdamW({len(self.params)} tensors, {bits}-bit moments, step {self.steps})"
