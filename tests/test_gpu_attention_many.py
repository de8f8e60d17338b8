"""Attention with more pieces of work than a launch's 32-bit count of threads has room for: 2^24 of 256."""
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu


def normal(device, dtype, *shape):
    return torch.randn(*shape, generator=torch.Generator(device=device).manual_seed(len(shape)), device=device).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_sequences(dtype, device):
    """2^20 and a few (sequence, head)s of one token each: every one sees itself."""
    shape = (2 ** 19 + 3, 1, 2, 16)
    q, v = normal(device, dtype, *shape), normal(device, dtype, *shape).flip(0)
    k, do = q.flip(3).contiguous(), v.flip(3).contiguous()
    o, kept = fm.attention_forward(q, k, v, keep=True)
    assert torch.equal(o, v)
    dq, dk, dv = fm.attention_pullback(do, q, k, v, o, kept)
    assert not dq.any() and not dk.any() and torch.equal(dv, do)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_unknown_lengths(dtype, device):
    """4200 short sequences of 64 heads, work laid out for as many tokens as there are in all: 17.7 million pieces."""
    lens = torch.arange(4200) % 4 + (torch.arange(4200) == 2000) * 150
    cu = torch.cat([torch.ones(1), 1 + lens.cumsum(0)]).int().to(device)
    shape = (8400, 64, 16)
    assert int(lens.sum()) < 8400 and 4200 * 64 * (8400 // 128 + 1) > 2 ** 24
    q, k, v, do = (normal(device, dtype, *shape).roll(i, 0) for i in range(4))
    results = []
    for lengths in ({}, dict(max_q=153, max_k=153)):
        args = dict(cu_q=cu, cu_k=cu, causal=True, **lengths)
        o, kept = fm.attention_forward(q, k, v, keep=True, **args)
        results.append((o, *fm.attention_pullback(do, q, k, v, o, kept, **args)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert all(t.any() for t in results[0])
