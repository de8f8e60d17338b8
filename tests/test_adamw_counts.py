"""The numbers of steps that AdamW gives its kernel, on the CPU: each tensor's own, and what the C
entries refuse of them before they launch anything."""
import numpy as np
import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import _lib, boundary, optim

OK, EINVAL, EUNSUP = _lib.FMS_OK, _lib.FMS_EINVAL, _lib.FMS_EUNSUPPORTED
RATES = (1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None)


def test_each_tensor_counts_its_own_steps(monkeypatch):
    seen = []
    monkeypatch.setattr(boundary, "require_device", lambda *ts: ts[0].device if ts else None)
    monkeypatch.setattr(boundary, "require_device_many", lambda *lists: torch.device("cpu"))
    monkeypatch.setattr(boundary, "stream_handle", lambda device: 0)
    monkeypatch.setattr(boundary, "adamw_step", lambda plan, device_plan, grads, dtypes, steps, *rest: seen.append(
        [int(n) if g else 0 for n, g in zip(steps, grads)]))
    opt = fm.AdamW([torch.ones(n) for n in (3, 5, 2)], step=[0, 4, 2])
    g = [torch.ones(n) for n in (3, 5, 2)]
    for grads in ([None, g[1], None], g, [g[0], None, g[2]], [None] * 3, g):
        opt.step(grads)
    assert seen == [[0, 5, 0], [1, 6, 3], [2, 0, 4], [3, 7, 5]]
    assert opt.tensor_steps == [3, 7, 5] and opt.steps == 8
    opt.steps = 10
    opt.step(g)
    assert seen[-1] == [11, 11, 11]


def test_entries_check_the_numbers_of_steps():
    L = _lib.lib()
    t = np.zeros(2, optim._ADAMW_ENTRY)
    t["p"] = t["m"] = t["v"] = 16
    t["n"] = [1, 2049]
    plan = np.zeros(L.fms_adamw_plan_bytes(2, t.ctypes.data), np.uint8)
    assert L.fms_adamw_plan(2, t.ctypes.data, plan.ctypes.data) == OK
    grads, dtypes = np.full(2, 16, np.uint64), np.array([0, 7], np.int32)

    def status(steps, plan=plan.ctypes.data, device_plan=16, rates=RATES):
        steps = None if steps is None else np.array(steps, np.int64)
        return L.fms_adamw_step_each(plan, device_plan, grads.ctypes.data, dtypes.ctypes.data,
                                     None if steps is None else steps.ctypes.data, *rates)

    assert status([1, 1]) == EUNSUP  # the second gradient's type
    for steps in (None, [0, 1], [-1, 1]):
        assert status(steps) == EINVAL
    assert status([1, 1], device_plan=None) == EINVAL and status([1, 1], plan=None) == EINVAL
    assert status([1, 1], rates=(1e-3, 1.0) + RATES[2:]) == EINVAL
    empty = np.zeros(16, np.uint8)
    assert L.fms_adamw_plan(0, None, empty.ctypes.data) == OK
    assert status(None, plan=empty.ctypes.data, device_plan=None) == OK


@pytest.mark.parametrize("bad", [[1], [1, -1], -1])
def test_numbers_of_steps_are_checked(monkeypatch, bad):
    monkeypatch.setattr(boundary, "require_device", lambda *ts: ts[0].device if ts else None)
    with pytest.raises((fm.ArgumentError, fm.DimensionMismatch)):
        fm.AdamW([torch.ones(2), torch.ones(2)], step=bad)
