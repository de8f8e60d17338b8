"""The encoder's raw calls check what they are given to write against what they read: an output of another type,
shape or device never reaches the library.  On the CPU, with arrays that say they are on a device and a library
that only counts its calls."""
import types

import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import boundary


@pytest.fixture
def calls(monkeypatch):
    """How often the library was called."""
    made = []
    functions = {n: (lambda *a, n=n: made.append(n) or 0)
                 for n in ("fms_attention", "fms_attention_pullback", "fms_head_rotary", "fms_head_rotary_pullback")}
    monkeypatch.setattr(boundary._lib, "lib", lambda: types.SimpleNamespace(**functions))
    monkeypatch.setattr(boundary, "_call_with_workspace", lambda fn, device, *args: fn(*args))
    monkeypatch.setattr(boundary, "stream_handle", lambda device: None)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: getattr(t, "at", 0))
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(torch.Tensor, "device", property(lambda t: torch.device("cuda", t.get_device())), raising=False)
    return made


Q, K, W = (2, 5, 4, 8), (2, 6, 2, 8), (8,)
HALF = dict(dtype=torch.float16)
OPTIONS = (None, None, None, None, 0, 0, 1.0, 0, -1)


def attention():
    arrays = {"o": torch.zeros(Q, **HALF), "top": torch.zeros(2, 2, 10), "rest": torch.zeros(Q, **HALF),
              "q": torch.zeros(Q, **HALF), "k": torch.zeros(K, **HALF), "v": torch.zeros(K, **HALF)}
    return arrays, lambda x: boundary.launch_attention(*x.values(), *OPTIONS), ("o", "rest"), ("k", "v")


def attention_pullback():
    shapes = dict(dq=Q, dk=K, dv=K, do=Q, o=Q, top=None, rest=Q, q=Q, k=K, v=K)
    arrays = {n: torch.zeros(2, 2, 10) if s is None else torch.zeros(s, **HALF) for n, s in shapes.items()}
    return (arrays, lambda x: boundary.attention_apply_pullback(*x.values(), *OPTIONS),
            ("dq", "dk", "dv", "do", "o", "rest"), ("k", "v"))


def rotary():
    k = (2, 5, 2, 8)
    arrays = {"q_out": torch.zeros(Q, **HALF), "k_out": torch.zeros(k, **HALF), "q": torch.zeros(Q, **HALF),
              "k": torch.zeros(k, **HALF)}
    return (arrays, lambda x: boundary.launch_head_rotary(*x.values(), torch.zeros(5, 8), None, None, None, 0, 0, 1e-6),
            ("q_out", "k_out"), ("k",))


def rotary_pullback():
    k = (2, 5, 2, 8)
    shapes = dict(dq=Q, dk=k, dwq=W, dwk=W, dq_out=Q, dk_out=k, q=Q, k=k)
    arrays = {n: torch.zeros(s, **HALF) for n, s in shapes.items()}
    w = torch.ones(W, **HALF)
    return (arrays, lambda x: boundary.head_rotary_apply_pullback(*x.values(), torch.zeros(5, 8), None, w, w, 0, 0, 1e-6),
            ("dq", "dk", "dwq", "dwk", "dq_out", "dk_out"), ("k",))


@pytest.mark.parametrize("made", [attention, attention_pullback, rotary, rotary_pullback])
def test_outputs_are_checked_against_inputs(made, calls):
    arrays, call, dense, heads = made()
    call(arrays)
    assert len(calls) == 1
    # (all that is written alike, and other than what is read)
    for others in [(n,) for n in dense] + [dense]:
        for change, error in ((lambda t: t.float(), fm.ArgumentError), (lambda t: t.bfloat16(), fm.ArgumentError),
                              (lambda t: t[..., :4].contiguous(), fm.DimensionMismatch),
                              (lambda t: t[:1].contiguous(), fm.DimensionMismatch),
                              (lambda t: torch.stack([t, t], -1)[..., 0], fm.ArgumentError)):
            with pytest.raises(error):
                call(arrays | {n: change(arrays[n]) for n in others})
        away = {n: arrays[n].clone() for n in others}
        for t in away.values():
            t.at = 1
        with pytest.raises(fm.ArgumentError):
            call(arrays | away)
    for n in heads:
        for part in (arrays[n][:1], arrays[n][:, :3], arrays[n][..., :4]):
            with pytest.raises(fm.DimensionMismatch):
                call(arrays | {n: part})
    assert len(calls) == 1
    # heads may lie as they like
    call(arrays | {n: torch.stack([arrays[n]] * 2, -2)[..., 0, :] for n in ("q", *heads)})
    assert len(calls) == 2
