"""AdamW's bias correction counts each tensor's own steps: one that had no gradient for a while, or
none at first, goes on from where it was.

Against torch's AdamW the bounds are those of the same formula in another order of operations; bit
for bit, such a tensor is stepped as by an optimiser that has it alone.
"""
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


def tensors(device, sizes, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    return [torch.randn(n, generator=g, device=device) for n in sizes]


def gradient(w, step):
    return torch.sin(w * (step + 1) + 0.3)


@pytest.mark.parametrize("active", [
    [lambda s: True, lambda s: s >= 7, lambda s: s % 3 == 0, lambda s: s < 2 or s > 8],
    [lambda s, i=i: s >= i for i in range(40)],  # more counts than a launch takes
], ids=["few", "many"])
def test_against_torch(device, active):
    w = tensors(device, [300 + 7 * i for i in range(len(active))])
    a, b = ([x.clone().requires_grad_() for x in w] for _ in range(2))
    ours, theirs = fm.AdamW(a, **HYPER), torch.optim.AdamW(b, foreach=False, fused=False, **HYPER)
    for s in range(len(active) + 4):
        for x, y, z, on in zip(a, b, w, active):
            x.grad, y.grad = (gradient(z, s), gradient(z, s)) if on(s) else (None, None)
        ours.step()
        theirs.step()
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [3, 500])
def test_as_if_alone(device, bits, count):
    """Tensor i has a gradient from step i % 5 on; 500 tensors are two launches."""
    w = tensors(device, [11 + i % 300 for i in range(count)])
    together, alone = ([x.clone() for x in w] for _ in range(2))
    opt = fm.AdamW(together, bits=bits, **HYPER)
    each = [fm.AdamW([x], bits=bits, **HYPER) for x in alone[:10]]
    for s in range(8):
        grads = [gradient(x, s) if s >= i % 5 else None for i, x in enumerate(w)]
        opt.step(grads)
        for i, o in enumerate(each):
            o.step([grads[i]])
    assert all(torch.equal(a, b) for a, b in zip(together, alone[:10]))
    assert opt.tensor_steps == [8 - i % 5 for i in range(count)] and opt.steps == 8


def test_going_on_from_counts(device):
    """An optimiser made from another's moments and counts goes on as that one would."""
    w = tensors(device, [300, 40])
    a, b = ([x.clone() for x in w] for _ in range(2))
    one = fm.AdamW(a, **HYPER)
    for s in range(3):
        one.step([gradient(w[0], s), gradient(w[1], s) if s == 2 else None])
    two = fm.AdamW(b, moments=([m.clone() for m in one.m], [v.clone() for v in one.v]),
                   step=one.tensor_steps, **HYPER)
    for x, y in zip(a, b):
        y.copy_(x)
    for opt in (one, two):
        opt.step([gradient(x, 3) for x in w])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert one.tensor_steps == two.tensor_steps == [4, 2] and one.steps == two.steps == 4
    two.steps = 9  # (all of them)
    assert two.tensor_steps == [9, 9]
    for bad in ([1], [1, -1], -1):
        with pytest.raises((fm.ArgumentError, fm.DimensionMismatch)):
            fm.AdamW(b, step=bad)
