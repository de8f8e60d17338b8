"""CPU checks of the encoder operators: status codes of the C entries and refusals of the Python layer, all
before any HIP call."""
import ctypes

import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import _lib

OK, EINVAL, EUNSUP = _lib.FMS_OK, _lib.FMS_EINVAL, _lib.FMS_EUNSUPPORTED


def attention(L, dtype=1, o=1, lse=None, rest=None, q=1, k=1, v=1, qmask=None, kmask=None, cu_q=None, cu_k=None,
              seqs=2, tq=8, tk=8, nq=0, nk=0, heads=4, kv_heads=2, dim=64, causal=0, window=-1, strides=None):
    st = None if strides is None else (ctypes.c_int64 * 9)(*strides)
    return L.fms_attention(dtype, o, lse, rest, q, k, v, st, qmask, kmask, cu_q, cu_k, seqs, tq, tk, nq, nk, heads,
                           kv_heads, dim, 0.125, causal, window, None)


def pullback(L, dtype=1, dq=1, dk=1, dv=1, dout=1, o=1, lse=1, rest=1, tq=8, tk=8, heads=4, dim=64):
    return L.fms_attention_pullback(dtype, dq, dk, dv, dout, o, lse, rest, 1, 1, 1, None, None, None, None, None, 2,
                                    tq, tk, 0, 0, heads, 2, dim, 0.125, 0, -1, None)


@pytest.mark.parametrize("args,expect", [
    (dict(dtype=9), EUNSUP), (dict(tq=-1), EINVAL), (dict(heads=3), EINVAL), (dict(kv_heads=0), EINVAL), (dict(heads=0), EINVAL),
    (dict(causal=2), EINVAL), (dict(window=-2), EINVAL), (dict(cu_q=1), EINVAL), (dict(cu_k=1), EINVAL),
    (dict(cu_q=1, cu_k=1, nq=-1), EINVAL), (dict(cu_q=1, cu_k=1, qmask=1), EINVAL), (dict(dim=129), EUNSUP),
    (dict(tq=1 << 29), EUNSUP), (dict(tk=1 << 29), EUNSUP), (dict(seqs=1 << 31), EUNSUP),
    (dict(heads=1 << 20, kv_heads=1 << 20), EUNSUP), (dict(tq=1 << 28, heads=8, kv_heads=1), EUNSUP),
    (dict(strides=[1] * 8 + [-1]), EINVAL), (dict(q=None), EINVAL), (dict(v=None), EINVAL), (dict(o=None), EINVAL),
    (dict(lse=1), EINVAL), (dict(rest=1), EINVAL), (dict(tq=0), OK), (dict(seqs=0), OK), (dict(heads=0, kv_heads=0), OK),
    (dict(dim=0), OK), (dict(seqs=1 << 20, tq=1 << 20), EUNSUP),
])
def test_attention_status(args, expect):
    assert attention(_lib.lib(), **args) == expect


@pytest.mark.parametrize("args,expect", [
    (dict(dtype=9), EUNSUP), (dict(dq=None), EINVAL), (dict(dk=None), EINVAL), (dict(dv=None), EINVAL),
    (dict(dout=None), EINVAL), (dict(o=None), EINVAL), (dict(lse=None), EINVAL), (dict(rest=None), EINVAL),
    (dict(dim=0), OK), (dict(tq=0, tk=0), OK),
])
def test_attention_pullback_status(args, expect):
    assert pullback(_lib.lib(), **args) == expect


def rotary(L, dtype=1, q_out=1, k_out=1, q=1, k=1, table=1, positions=None, id_bytes=4, placed=1, kind=0, pairing=0,
           seqs=2, tokens=5, heads=4, kv_heads=2, dim=64, turned=64, rows=5):
    return L.fms_head_rotary(dtype, q_out, k_out, q, k, None, table, positions, id_bytes, placed, None, None, kind,
                             pairing, 1e-6, seqs, tokens, heads, kv_heads, dim, turned, rows, None)


@pytest.mark.parametrize("args,expect", [
    (dict(dtype=3), EUNSUP), (dict(kind=2), EINVAL), (dict(pairing=-1), EINVAL), (dict(dim=63), EINVAL),
    (dict(turned=66), EINVAL), (dict(turned=7), EINVAL), (dict(rows=4), EINVAL), (dict(dim=514), EUNSUP),
    (dict(positions=1, id_bytes=2), EINVAL), (dict(positions=1, placed=3), EINVAL), (dict(q=None), EINVAL),
    (dict(k=None), EINVAL), (dict(table=None), EINVAL), (dict(q_out=None), EINVAL), (dict(k_out=None), EINVAL),
    (dict(tokens=0), OK), (dict(seqs=0), OK), (dict(heads=0, kv_heads=0, q=None, k=None), OK), (dict(seqs=-1), EINVAL),
    (dict(seqs=1 << 31), EUNSUP),
])
def test_rotary_status(args, expect):
    assert rotary(_lib.lib(), **args) == expect


@pytest.mark.parametrize("call,expect", [
    (lambda L: L.fms_embed_tokens(9, 1, 1, 4, 1, 1.0, 4, 8, 8, None), EUNSUP),
    (lambda L: L.fms_embed_tokens(1, 1, 1, 2, 1, 1.0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_embed_tokens(1, 1, 1, 4, 1, 1.0, -1, 8, 8, None), EINVAL),
    (lambda L: L.fms_embed_tokens(1, 1, None, 4, 1, 1.0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_embed_tokens(1, 1, 1, 4, None, 1.0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_embed_tokens(1, None, 1, 4, 1, 1.0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_embed_tokens(1, 1, 1, 4, 1, 1.0, 1 << 31, 8, 8, None), EUNSUP),
    (lambda L: L.fms_embed_tokens(1, None, None, 4, None, 1.0, 0, 8, 8, None), OK),
    (lambda L: L.fms_embed_tokens_pullback(1, None, 1, 1, 4, 1.0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_embed_tokens_pullback(1, 1, None, 1, 4, 1.0, 4, 8, 8, None), EINVAL),
    (lambda L: L.fms_embed_tokens_pullback(1, None, None, 1, 4, 1.0, 4, 0, 8, None), OK),
    (lambda L: L.fms_embed_tokens_pullback(1, 1, 1, 1, 4, 1.0, 4, (1 << 31) - 1, 8, None), EUNSUP),
])
def test_embed_status(call, expect):
    assert call(_lib.lib()) == expect


def test_host_arrays_are_refused():
    q, ids, table = torch.zeros(2, 4, 2, 32), torch.ones(3, dtype=torch.int32), torch.zeros(4, 32)
    for call in (lambda: fm.attention_forward(q, q, q), lambda: fm.attention(q, q, q),
                 lambda: fm.head_rotary_forward(q, q, table), lambda: fm.embed_tokens_forward(ids, torch.zeros(5, 8)),
                 lambda: fm.embed_tokens_pullback(torch.zeros(3, 8), ids, 5)):
        with pytest.raises(fm.ArgumentError):
            call()


def test_heads_are_refused():
    """Key heads that no query head shares: their gradients would be nobody's."""
    for h, hk in ((0, 2), (2, 0), (3, 2)):
        with pytest.raises(fm.DimensionMismatch):
            fm.attention_forward(torch.zeros(1, 4, h, 32), torch.zeros(1, 5, hk, 32), torch.zeros(1, 5, hk, 32))
