"""CPU checks of the token-block operators: status codes of the C entries and refusals of the
Python layer, all before any HIP call."""
import numpy as np
import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import _lib, optim

OK, EINVAL, EUNSUP = _lib.FMS_OK, _lib.FMS_EINVAL, _lib.FMS_EUNSUPPORTED
NAN = float("nan")


def adamw(L, plan=0, step=1, beta1=0.9, beta2=0.999, eps=1e-8):
    """fms_adamw_step over an empty plan."""
    empty = np.zeros(16, np.uint8)
    assert L.fms_adamw_plan_bytes(0, None) == 16 and L.fms_adamw_plan(0, None, empty.ctypes.data) == OK
    return L.fms_adamw_step(empty.ctypes.data if plan == 0 else plan, None, None, None, step, 1e-3, beta1,
                            beta2, eps, 0.0, 1.0, None)


@pytest.mark.parametrize("call,expect", [
    # gated_ffn: dtype, activation, sizes, NULL arrays, empty calls, sizes past 32-bit offsets
    (lambda L: L.fms_gated_ffn(9, 1, 1, 1, 1, 0, 4, 8, 8, None), EUNSUP),
    (lambda L: L.fms_gated_ffn(1, 1, 1, 1, 1, 3, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_gated_ffn(1, 1, 1, 1, 1, -1, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_gated_ffn(1, 1, 1, 1, 1, 0, -4, 8, 8, None), EINVAL),
    (lambda L: L.fms_gated_ffn(1, None, 1, 1, 1, 0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_gated_ffn(1, 1, None, 1, 1, 0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_gated_ffn(1, 1, 1, 1, None, 0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_gated_ffn(1, None, None, 1, 1, 0, 0, 8, 8, None), OK),
    (lambda L: L.fms_gated_ffn(1, None, 1, None, None, 0, 4, 8, 0, None), OK),
    (lambda L: L.fms_gated_ffn(0, 1, 1, 1, 1, 0, 4, 1 << 21, 8, None), EUNSUP),
    (lambda L: L.fms_gated_ffn(0, 1, 1, 1, 1, 0, 1 << 31, 8, 8, None), EUNSUP),
    (lambda L: L.fms_gated_ffn(0, 1, 1, 1, 1, 0, 1 << 30, 8, 4096, None), EUNSUP),
    (lambda L: L.fms_gated_ffn_pullback(1, 1, 1, None, 1, 1, 1, 1, 0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_gated_ffn_pullback(1, 1, 1, 1, None, 1, 1, 1, 0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_gated_ffn_pullback(1, None, None, None, 1, 1, 1, 1, 0, 4, 8, 8, None), OK),
    (lambda L: L.fms_gated_ffn_pullback(1, None, None, None, None, None, None, None, 0, 0, 0, 0, None), OK),
    # block_norm: kind, gates that do not divide the rows, missing outputs, width, empty calls
    (lambda L: L.fms_block_norm(9, 1, 1, 1, 1, None, None, 1, 0, 1.0, 1e-6, 4, 8, 4, None), EUNSUP),
    (lambda L: L.fms_block_norm(0, 1, 1, 1, 1, None, None, 1, 2, 1.0, 1e-6, 4, 8, 4, None), EINVAL),
    (lambda L: L.fms_block_norm(0, 1, 1, 1, 1, 1, None, 1, 0, 1.0, 1e-6, 4, 8, 3, None), EINVAL),
    (lambda L: L.fms_block_norm(0, 1, 1, 1, 1, 1, None, 1, 0, 1.0, 1e-6, 4, 8, 0, None), EINVAL),
    (lambda L: L.fms_block_norm(0, 1, 1, 1, None, 1, None, 1, 0, 1.0, 1e-6, 4, 8, 4, None), EINVAL),
    (lambda L: L.fms_block_norm(0, None, 1, 1, 1, None, None, 1, 0, 1.0, 1e-6, 4, 8, 4, None), EINVAL),
    (lambda L: L.fms_block_norm(0, 1, None, 1, 1, None, None, 1, 0, 1.0, 1e-6, 4, 8, 4, None), EINVAL),
    (lambda L: L.fms_block_norm(0, 1, 1, None, 1, None, None, 1, 0, 1.0, 1e-6, 4, 8, 4, None), EINVAL),
    (lambda L: L.fms_block_norm(0, 1, 1, 1, 1, None, None, 1, 0, 1.0, 1e-6, 4, 16385, 4, None), EUNSUP),
    (lambda L: L.fms_block_norm(0, None, None, None, None, None, None, None, 0, 1.0, 1e-6, 0, 8, 1, None), OK),
    (lambda L: L.fms_block_norm_pullback(0, 1, 1, None, None, None, None, 1, 1, 1, None, None, None, 0,
                                         1.0, 1e-6, 4, 8, 4, None), EINVAL),  # dn without wpre
    (lambda L: L.fms_block_norm_pullback(0, None, 1, None, None, None, 1, None, 1, 1, None, None, None, 0,
                                         1.0, 1e-6, 4, 8, 4, None), EINVAL),  # no dx
    (lambda L: L.fms_block_norm_pullback(0, 1, None, None, None, None, 1, None, 1, 1, None, None, None, 0,
                                         1.0, 1e-6, 4, 8, 4, None), EINVAL),  # no df
    (lambda L: L.fms_block_norm_pullback(0, 1, 1, None, None, None, 1, None, 1, 1, 1, None, None, 0,
                                         1.0, 1e-6, 4, 8, 4, None), EINVAL),  # no dgate
    # AdamW: plan, step, hyperparameters
    (lambda L: L.fms_adamw_plan(-1, None, 1), EINVAL),
    (lambda L: L.fms_adamw_plan(1, None, 1), EINVAL),
    (lambda L: L.fms_adamw_plan(0, None, None), EINVAL),
    (lambda L: adamw(L, plan=None), EINVAL),
    (lambda L: adamw(L, step=0), EINVAL),
    (lambda L: adamw(L, beta1=1.0), EINVAL),
    (lambda L: adamw(L, beta2=NAN), EINVAL),
    (lambda L: adamw(L, eps=-1.0), EINVAL),
    (lambda L: adamw(L), OK),  # a plan of nothing
    (lambda L: L.fms_moment_values(-1, None, None), EINVAL),
    (lambda L: L.fms_moment_values(2, None, None), EINVAL),
    (lambda L: L.fms_moment_values(0, None, None), OK),
])
def test_status_codes(call, expect):
    assert call(_lib.lib()) == expect


def test_adamw_plans():
    """Entries are checked, and a plan holds them with the tensor of each 2048 elements."""
    L = _lib.lib()

    def status(**entry):
        t = np.zeros(1, optim._ADAMW_ENTRY)
        for k, v in (dict(p=1, m=1, v=1, n=8) | entry).items():
            t[k] = v
        plan = np.zeros(4096, np.uint8)
        s = L.fms_adamw_plan(1, t.ctypes.data, plan.ctypes.data)
        assert (L.fms_adamw_plan_bytes(1, t.ctypes.data) < 0) == (s != OK)
        return s

    assert status(p_dtype=9) == EUNSUP and status(p_dtype=-1) == EUNSUP
    assert status(n=-1) == EINVAL and status(p=0) == EINVAL and status(v=0) == EINVAL
    assert status(m_scale=1) == EINVAL  # one scale without the other
    assert status(n=(1 << 33) + 1) == EUNSUP
    assert status(n=0, p=0, m=0, v=0) == OK

    t = np.zeros(4, optim._ADAMW_ENTRY)
    t["p"] = t["m"] = t["v"] = 16
    t["n"] = [1, 0, 2049, 4096]
    n = L.fms_adamw_plan_bytes(4, t.ctypes.data)
    assert n == 16 + 4 * 72 + 5 * 4
    plan = np.zeros(n + 4, np.uint8)
    assert L.fms_adamw_plan(4, t.ctypes.data, plan.ctypes.data) == OK
    assert plan[:16].view(np.int64).tolist() == [4, 5] and not plan[n:].any()
    assert plan[16 + 4 * 72:n].view(np.int32).tolist() == [0, 2, 2, 3, 3]
    entries = plan[16:16 + 4 * 72].view(np.int64).reshape(4, 9)
    assert entries[:, 8].tolist() == [0, 1, 1, 3] and entries[:, 6].tolist() == [1, 0, 2049, 4096]
    # a step refuses gradients of unknown types and missing arrays before it launches
    grads, dtypes = np.full(4, 16, np.uint64), np.array([0, 1, 7, 2], np.int32)
    args = (1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None)
    assert L.fms_adamw_step(plan.ctypes.data, 16, grads.ctypes.data, dtypes.ctypes.data, *args) == EUNSUP
    assert L.fms_adamw_step(plan.ctypes.data, None, grads.ctypes.data, dtypes.ctypes.data, *args) == EINVAL
    assert L.fms_adamw_step(plan.ctypes.data, 16, None, dtypes.ctypes.data, *args) == EINVAL


def test_table_layout_is_the_headers():
    """fms_adamw_tensor: six pointers, n, a dtype; fms_moment8: three pointers, n, a flag."""
    assert optim._ADAMW_ENTRY.itemsize == 64 and optim._ADAMW_ENTRY.fields["n"][1] == 48
    assert optim._MOMENT_ENTRY.itemsize == 40


def test_host_arrays_and_bad_arguments_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(fm.ArgumentError):
        fm.gated_ffn(x, w, w)
    with pytest.raises(fm.ArgumentError):
        fm.gated_ffn_forward(x, w, w, act="relu")
    with pytest.raises(fm.DimensionMismatch):
        fm.gated_ffn_forward(x, w[0], w)
    with pytest.raises(fm.DimensionMismatch):
        fm.gated_ffn_pullback(torch.zeros(4, 5), x, w, w)
    with pytest.raises(fm.ArgumentError):
        fm.block_norm(x, pre_weight=torch.ones(8))
    with pytest.raises(fm.ArgumentError):
        fm.block_norm(x)
    with pytest.raises(fm.ArgumentError):
        fm.block_norm(x, gate=torch.ones(8), pre_weight=torch.ones(8))
    with pytest.raises(fm.DimensionMismatch):
        fm.block_norm(x, x, gate=torch.ones(3, 8))
    with pytest.raises(fm.ArgumentError):
        fm.AdamW([x])
    with pytest.raises(fm.ArgumentError):
        fm.Moment8(torch.zeros(8), torch.zeros(1))
    with pytest.raises(fm.DimensionMismatch):
        fm.Moment8(torch.zeros(257, dtype=torch.int8), torch.zeros(1))
