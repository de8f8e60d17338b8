"""Where AdamW's arrays lie, on the CPU: what a step's plan tells the kernel to read and write,
with the launch itself replaced.  A plan holds addresses, so every one of them must belong to an
array that the optimiser still has, wherever that has been moved."""
import numpy as np
import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import boundary, optim

ENTRY = np.dtype([(k, optim._ADAMW_ENTRY.fields[k][0].str) for k in optim._ADAMW_ENTRY.names] + [("first", "i8")])


@pytest.fixture
def launches(monkeypatch):
    """The plans' entries of the steps launched, and the gradients' addresses."""
    seen = []

    def require(*ts):
        ts = [t for t in ts if t is not None]
        for t in ts:
            if not isinstance(t, torch.Tensor):
                raise fm.ArgumentError("not a tensor")
            if not t.is_contiguous():
                raise fm.ArgumentError("FlashMaxSim device arrays must be dense (contiguous)")
        return ts[0].device if ts else None

    def launch(plan, device_plan, grads, *rest):
        assert np.array_equal(plan, device_plan.numpy())
        count = int(plan[:8].view(np.int64)[0])
        seen.append((plan[16:16 + count * ENTRY.itemsize].view(ENTRY).copy(), grads.copy()))

    monkeypatch.setattr(boundary, "require_device", require)
    monkeypatch.setattr(boundary, "require_device_many", lambda *ls: require(*[t for l in ls for t in l]))
    monkeypatch.setattr(boundary, "stream_handle", lambda device: 0)
    monkeypatch.setattr(boundary, "adamw_step", launch)
    return seen


SIZES = [700, 3, 256]


def optimiser(bits, **kw):
    params = [torch.randn(n).bfloat16() for n in SIZES]
    return fm.AdamW(params, bits=bits, masters=True, **kw), [torch.randn(n).bfloat16() for n in SIZES]


def arrays(opt, i):
    """{name in the plan: the optimiser's array} of tensor i."""
    m, v = opt.m[i], opt.v[i]
    found = {"p": opt.params[i], "master": opt.masters[i]}
    if isinstance(m, fm.Moment8):
        return found | {"m": m.codes, "v": v.codes, "m_scale": m.scales, "v_scale": v.scales}
    return found | {"m": m, "v": v}


def check(entries, opt):
    for i, e in enumerate(entries):
        for name, t in arrays(opt, i).items():
            assert e[name] == t.data_ptr(), (i, name)
        assert e["n"] == opt.params[i].numel()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("again", [False, True])
def test_a_moved_array_is_stepped_where_it_lies(launches, bits, again):
    """Each array in turn given new memory, as restoring or offloading does, before the first step
    and between steps."""
    names = ["p", "master", "m", "v"] + (["m_scale", "v_scale"] if bits == 8 else [])
    opt, grads = optimiser(bits)
    if again:
        opt.step(grads)
    for i in range(len(SIZES)):
        for name in names:
            t = arrays(opt, i)[name]
            old = t.data_ptr()
            keep = t.data  # (its memory is not given out again)
            t.data = t.data.clone()
            opt.step(grads)
            assert launches[-1][0][i][name] != old
            check(launches[-1][0], opt)
            del keep


def test_new_codes_of_a_moment(launches):
    """A Moment8 given other arrays: the step and moment_values use the same ones."""
    opt, grads = optimiser(8)
    opt.step(grads)
    opt.m[0].codes = opt.m[0].codes.clone()
    opt.v[1].scales = opt.v[1].scales.clone()
    opt.step(grads)
    check(launches[-1][0], opt)
    for codes, error in ((torch.zeros(699, dtype=torch.int8), fm.DimensionMismatch),
                         (torch.zeros(700, dtype=torch.uint8), fm.ArgumentError)):
        kept = opt.m[0].codes
        opt.m[0].codes = codes
        with pytest.raises(error):
            opt.step(grads)
        opt.m[0].codes = kept
    assert len(launches) == 2 and opt.steps == 2
    opt.step(grads)
    check(launches[-1][0], opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_given_moments_are_held(launches, bits):
    """The optimiser works on the memory that it was given, whatever its giver does with the
    tensors afterwards."""
    params = [torch.randn(n) for n in SIZES]
    m, v = ([fm.Moment8.zeros(p, s) if bits == 8 else torch.zeros_like(p) for p in params] for s in (True, False))
    masters = [torch.zeros_like(p) for p in params]
    given = [t for x in m + v for t in ((x.codes, x.scales) if bits == 8 else (x,))] + masters
    where = [t.data_ptr() for t in given]
    opt = fm.AdamW(params, moments=(m, v), masters=masters)
    for t in given:
        t.data = torch.ones_like(t)
    later = [torch.empty_like(t) for t in given]  # (takes what was free)
    opt.step([torch.randn(n) for n in SIZES])
    entries = launches[-1][0]
    check(entries, opt)
    names = ("m", "v", "master") + (("m_scale", "v_scale") if bits == 8 else ())
    used = {int(e[k]) for e in entries for k in names}
    assert used == set(where)
    assert not used & {t.data_ptr() for t in later + given}


@pytest.mark.parametrize("bits", [32, 8])
def test_moved_arrays_are_checked(launches, bits):
    """Moved to where it cannot be stepped: refused, step after step, and no step is counted."""
    opt, grads = optimiser(bits)
    opt.step(grads)
    t = arrays(opt, 0)["m"]
    good = t.data
    for bad, error in ((torch.zeros(699, dtype=t.dtype), fm.DimensionMismatch),
                       (torch.zeros(1400, dtype=t.dtype)[::2], fm.ArgumentError),
                       (opt.masters[0].data.view(torch.int8)[:700] if bits == 8 else opt.masters[0].data,
                        fm.ArgumentError)):
        t.data = bad
        for _ in range(2):
            with pytest.raises(error):
                opt.step(grads)
        t.data = good
    assert opt.steps == 1 and len(launches) == 1
    opt.step(grads)
    check(launches[-1][0], opt)


def test_state_is_the_optimisers(launches):
    """m, v and masters are changed in place, not replaced."""
    opt, _ = optimiser(32)
    for name in ("m", "v", "masters"):
        with pytest.raises(AttributeError):
            setattr(opt, name, getattr(opt, name))


def test_moved_float_moments_by_their_values(launches):
    """moment_values() of 32-bit moments are the moments themselves: moving those counts too."""
    opt, grads = optimiser(32)
    (m, _) = opt.moment_values()
    opt.step(grads)
    m[0].data = m[0].data.clone()
    opt.step(grads)
    check(launches[-1][0], opt)
