"""Attention where a query sees one key: its weight is one, so the output is that key's value and the gradients
of the query and the key are zero.  Exactly: nothing is rounded on the way, and an optimiser that divides by a
gradient's size would make steps out of what is left of a rounding."""
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(shape_q, shape_k, dtype, device, size=1.0):
    g = torch.Generator(device=device).manual_seed(shape_q[0] * 1000 + shape_k[-3])
    normal = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    return [t.to(dtype) for t in (normal(*shape_q) * size, normal(*shape_k) * size, normal(*shape_k), normal(*shape_q))]


def both(q, k, v, do, **args):
    o, kept = fm.attention_forward(q, k, v, keep=True, **args)
    assert torch.equal(o, fm.attention_forward(q, k, v, **args))
    return (o, *fm.attention_pullback(do, q, k, v, o, kept, **args))


def shared(v, heads):
    """The values that each query head sees."""
    return v.repeat_interleave(heads // v.shape[-2], -2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Tq,H,Hk,d", [(63, 13, 18, 9, 77), (3, 1, 4, 4, 64), (2, 200, 2, 1, 128), (5, 40, 3, 3, 32),
                                         (1, 70, 8, 2, 16)])
def test_one_key(dtype, B, Tq, H, Hk, d, device):
    q, k, v, do = inputs((B, Tq, H, d), (B, 1, Hk, d), dtype, device)
    o, dq, dk, _ = both(q, k, v, do)
    assert torch.equal(o, shared(v, H).expand(q.shape))
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1.0, 5.0, 100.0])
@pytest.mark.parametrize("H,Hk,d", [(4, 4, 64), (6, 2, 128), (2, 2, 40)])
def test_no_window(dtype, size, H, Hk, d, device):
    """A window of 0: every token sees itself."""
    q, k, v, do = inputs((2, 300, H, d), (2, 300, Hk, d), dtype, device, size)
    o, dq, dk, _ = both(q, k, v, do, window=0)
    assert torch.equal(o, shared(v, H))
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_ragged_tokens(dtype, device):
    """Sequences of one token, and longer ones in a window of 0."""
    lens = torch.tensor([1, 1, 0, 90, 1, 200, 1])
    cu = torch.cat([torch.ones(1), 1 + lens.cumsum(0)]).int().to(device)
    n = int(lens.sum())
    q, k, v, do = inputs((n, 4, 64), (n, 2, 64), dtype, device)
    o, dq, dk, _ = both(q, k, v, do, cu_q=cu, cu_k=cu, max_q=200, max_k=200, window=0)
    assert torch.equal(o, shared(v, 4))
    assert not dq.any() and not dk.any()
    ones = torch.arange(1, n + 2, dtype=torch.int32, device=device)
    o, dq, dk, _ = both(q, k, v, do, cu_q=ones, cu_k=ones, max_q=1, max_k=1)
    assert torch.equal(o, shared(v, 4))
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Tq,Tk,H,Hk,d", [(150, 170, 4, 2, 64), (1, 5000, 4, 1, 128), (2, 1000, 2, 2, 48), (130, 1100, 1, 1, 32)])
def test_mask_leaves_one(dtype, Tq, Tk, H, Hk, d, device):
    """Among them calls whose few rows' keys are split among workgroups and joined."""
    q, k, v, do = inputs((2, Tq, H, d), (2, Tk, Hk, d), dtype, device)
    left = torch.tensor([Tk // 3, Tk - 1], device=device)
    mask = torch.arange(Tk, device=device) == left[:, None]
    o, dq, dk, _ = both(q, k, v, do, kmask=mask)
    assert torch.equal(o, shared(v[torch.arange(2, device=device), left][:, None], H).expand(q.shape))
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [None, -0.3])
def test_first_of_a_causal_sequence(dtype, scale, device):
    """The first token sees itself alone, others see more."""
    q, k, v, do = inputs((40, 30, 2, 64), (40, 30, 2, 64), dtype, device)
    o, dq, _, _ = both(q, k, v, do, causal=True, scale=scale)
    assert torch.equal(o[:, 0], v[:, 0])
    assert not dq[:, 0].any() and dq[:, 1:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1.0, 30.0, 100.0])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("scale", [None, 2.0, -0.7])
def test_value_gradients(dtype, size, d, scale, device):
    """Each key seen by one query alone: dv is that query's cotangent, however large the score."""
    q, k, v, do = inputs((2, 200, 2, d), (2, 200, 2, d), dtype, device, size)
    assert torch.equal(both(q, k, v, do, window=0, scale=scale)[3], do)
    q, k, v, do = inputs((30, 1, 3, d), (30, 1, 3, d), dtype, device, size)
    assert torch.equal(both(q, k, v, do, scale=scale)[3], do)
