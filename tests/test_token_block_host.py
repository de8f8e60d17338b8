"""CPU checks of the token-block operators: status codes of the C entries and refusals of the
Python layer, all before any HIP call."""
import ctypes

import numpy as np
import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import _lib, optim

OK, EINVAL, EUNSUP = _lib.FMS_OK, _lib.FMS_EINVAL, _lib.FMS_EUNSUPPORTED
NAN = float("nan")


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
    # AdamW: table, step, hyperparameters
    (lambda L: L.fms_adamw_step(-1, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None), EINVAL),
    (lambda L: L.fms_adamw_step(1, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None), EINVAL),
    (lambda L: L.fms_adamw_step(0, None, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None), EINVAL),
    (lambda L: L.fms_adamw_step(0, None, 1, 1e-3, 1.0, 0.999, 1e-8, 0.0, 1.0, None), EINVAL),
    (lambda L: L.fms_adamw_step(0, None, 1, 1e-3, 0.9, NAN, 1e-8, 0.0, 1.0, None), EINVAL),
    (lambda L: L.fms_adamw_step(0, None, 1, 1e-3, 0.9, 0.999, -1.0, 0.0, 1.0, None), EINVAL),
    (lambda L: L.fms_adamw_step(0, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None), OK),
    (lambda L: L.fms_moment_values(-1, None, None), EINVAL),
    (lambda L: L.fms_moment_values(2, None, None), EINVAL),
    (lambda L: L.fms_moment_values(0, None, None), OK),
])
def test_status_codes(call, expect):
    assert call(_lib.lib()) == expect


def test_adamw_table_entries_are_checked():
    def status(**entry):
        t = np.zeros(1, optim._ADAMW_ENTRY)
        for k, v in (dict(p=1, g=1, m=1, v=1, n=8) | entry).items():
            t[k] = v
        return _lib.lib().fms_adamw_step(1, t.ctypes.data, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None)

    assert status(p_dtype=9) == EUNSUP and status(g_dtype=-1) == EUNSUP
    assert status(n=-1) == EINVAL and status(g=0) == EINVAL and status(v=0) == EINVAL
    assert status(m_scale=1) == EINVAL  # one scale without the other
    assert status(n=(1 << 33) + 1) == EUNSUP
    assert status(n=0, p=0, g=0, m=0, v=0) == OK


def test_table_layout_is_the_headers():
    """fms_adamw_tensor: seven pointers, n, two dtypes; fms_moment8: three pointers, n, a flag."""
    class Entry(ctypes.Structure):
        _fields_ = [(k, ctypes.c_void_p) for k in ("p", "g", "m", "v", "master", "m_scale", "v_scale")] + [
            ("n", ctypes.c_int64), ("p_dtype", ctypes.c_int32), ("g_dtype", ctypes.c_int32)]

    assert optim._ADAMW_ENTRY.itemsize == ctypes.sizeof(Entry) == 72
    assert all(optim._ADAMW_ENTRY.fields[k][1] == getattr(Entry, k).offset for k, _ in Entry._fields_)
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
