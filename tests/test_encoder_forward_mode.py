"""Forward-mode derivatives are refused by the encoder's verbs: none of them returns a result without a tangent.
Host arrays, the launches left out."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import flashmaxsim as fm
from flashmaxsim import boundary


@pytest.fixture
def launched(monkeypatch):
    calls = []
    for name in ("launch_attention", "launch_head_rotary", "launch_embed_tokens"):
        monkeypatch.setattr(boundary, name, lambda *a, name=name: calls.append(name))
    return calls


def verbs():
    q, k, v = torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 2, 8), torch.zeros(2, 5, 2, 8)
    w, table = torch.ones(8), torch.zeros(5, 8)
    ids = torch.ones(3, dtype=torch.int32)
    return {"attention": (lambda *x: fm.attention(*x), [q, k, v]),
            "head_rotary": (lambda q, k, a, b: fm.head_rotary(q, k, table, q_weight=a, k_weight=b), [q, k, w, w]),
            "embed_tokens": (lambda w: fm.embed_tokens(ids, w), [torch.zeros(7, 8)])}


@pytest.mark.parametrize("name", verbs())
def test_duals_are_refused(name, launched):
    call, arrays = verbs()[name]
    for i, t in enumerate(arrays):
        with fw.dual_level(), pytest.raises(NotImplementedError):
            call(*arrays[:i], fw.make_dual(t, torch.ones_like(t)), *arrays[i + 1:])
        with fw.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
            call(*arrays[:i], fw.make_dual(t, torch.ones_like(t)), *arrays[i + 1:])
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, tuple(arrays), tuple(map(torch.ones_like, arrays)))


@pytest.mark.parametrize("name", verbs())
def test_other_tensors_are_not(name, launched):
    """Inside a level, what has no tangent is computed as outside."""
    call, arrays = verbs()[name]
    with fw.dual_level():
        call(*arrays)
    assert len(launched) == 1
