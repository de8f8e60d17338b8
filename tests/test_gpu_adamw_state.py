"""AdamW's moments and masters on the GPU: moved between steps, and let go after a step on another
stream than their own."""
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


def make(device, sizes, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    return ([torch.randn(n, generator=g, device=device).to(dtype) for n in sizes],
            [torch.randn(n, generator=g, device=device).to(dtype) for n in sizes])


def arrays(opt):
    for m in opt.m + opt.v:
        yield from (m.codes, m.scales) if isinstance(m, fm.Moment8) else (m,)
    yield from (w for w in opt.masters if w is not None)


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_and_masters_may_move(device, bits):
    """Every one of them given new memory between steps: the steps go on there, and leave the old
    memory as it was."""
    params, grads = make(device, [3000, 5, 257])
    other = [p.clone() for p in params]
    opt, ref = (fm.AdamW(p, bits=bits, masters=True, **HYPER) for p in (params, other))
    for _ in range(3):
        opt.step(grads)
        ref.step(grads)
        old = [t.data for t in arrays(opt)]
        kept = [t.clone() for t in old]
        for t in arrays(opt):
            t.data = t.data.clone()
        opt.step(grads)
        ref.step(grads)
        assert all(torch.equal(a, b) for a, b in zip(params, other))
        assert all(torch.equal(a, b) for a, b in zip(arrays(opt), arrays(ref)))
        assert all(torch.equal(a, b) for a, b in zip(old, kept))


def test_restored_by_copying(device):
    """Moments and masters copied into are gone on from."""
    params, grads = make(device, [3000, 5])
    one = fm.AdamW(params, bits=8, masters=True, **HYPER)
    one.step(grads)
    saved, p = [t.clone() for t in arrays(one)], [p.clone() for p in params]
    one.step(grads)
    two = fm.AdamW(p, bits=8, masters=True, step=1, **HYPER)
    for t, s in zip(arrays(two), saved):
        t.copy_(s)
    two.step(grads)
    assert all(torch.equal(a, b) for a, b in zip(params, p))
    assert all(torch.equal(a, b) for a, b in zip(arrays(one), arrays(two)))


@pytest.mark.parametrize("bits", [32, 8])
def test_own_memory_after_a_step_on_another_stream(device, bits):
    """What the optimiser made for itself is not given out again before a step on a stream of
    its own is through, though the optimiser is dropped."""
    params, grads = make(device, [70001] * 4)
    other = [p.clone() for p in params]
    fm.AdamW(params, bits=bits, masters=True, **HYPER).step(grads)
    opt = fm.AdamW(other, bits=bits, masters=True, **HYPER)
    shapes = [(t.shape, t.dtype) for t in arrays(opt)]
    at = {t.data_ptr() for t in arrays(opt)}
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    busy = torch.ones(4096, 4096, device=device)
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy @ busy * 2.0 ** -12
        opt.step(grads)
    del opt
    later = [torch.zeros(s, dtype=d, device=device) for s, d in shapes * 2]
    assert not at & {t.data_ptr() for t in later}
    torch.cuda.current_stream(device).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(params, other))
    assert not any(t.any() for t in later)
