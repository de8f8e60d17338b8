"""The AdamW step on the GPU against its formula in 64 bits; 8-bit moments against their
definition, bit for bit, from IEEE fp32 arithmetic on the CPU."""
import math

import numpy as np
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SIZES = [1, 2, 7, 8, 255, 256, 257, 2047, 2048, 2049, 5000, 70001]
HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
f32 = np.float32


def rows256(x):
    return np.pad(x, (0, -len(x) % 256)).reshape(-1, 256)


def encode(x, signed):
    """Codes and scales of fp32 values by the definition."""
    r = rows256(x)
    top = np.abs(r).max(1, keepdims=True)
    scale = np.where(top < np.finfo(f32).tiny, f32(0), top)
    with np.errstate(divide="ignore"):
        inv = np.where(scale == 0, f32(0), f32(1) / top)
    q = np.abs(r) * inv
    if signed:
        c = np.sign(r) * np.rint(np.sqrt(q) * f32(127))
    else:
        c = np.rint(np.sqrt(np.sqrt(q)) * f32(255))
        c = np.where((q > 0) & (c < 1), 1, c)
    return c.reshape(-1)[:len(x)].astype(np.int8 if signed else np.uint8), scale.reshape(-1)


def decode(c, scale):
    a = np.repeat(scale, 256)[:len(c)]
    if c.dtype == np.int8:
        t = c.astype(f32) * f32(1 / 127)
        return np.sign(c).astype(f32) * (t * t) * a
    t = c.astype(f32) * f32(1 / 255)
    t = t * t
    return t * t * a


def step32(p, g, m, v, step, lr, betas, eps, weight_decay, grad_scale=1.0):
    """The step in fp32, each operation rounded by itself."""
    b1, b2 = betas
    g = g * f32(grad_scale)
    m = m * f32(b1) + g * f32(1 - b1)
    v = v * f32(b2) + g * g * f32(1 - b2)
    den = np.sqrt(v) * f32(1 / math.sqrt(1 - b2 ** step)) + f32(eps)
    p = p * f32(1 - lr * weight_decay) - m / den * f32(lr / (1 - b1 ** step))
    return p, m, v


def tensors(device, dtype, gdtype=None, sizes=SIZES, offset=0, seed=0):
    rng = np.random.default_rng(seed)

    def dev(x, d):
        t = torch.empty(len(x) + offset, dtype=d, device=device)[offset:]
        return t.copy_(torch.from_numpy(x))

    p = [rng.standard_normal(n, dtype=f32) * f32(0.1) for n in sizes]
    g = [rng.standard_normal(n, dtype=f32) * f32(10.0 ** rng.integers(-4, 1)) for n in sizes]
    return [dev(x, dtype) for x in p], [dev(x, gdtype or dtype) for x in g]


def np32(t):
    return t.detach().float().cpu().numpy()


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("dtype,gdtype", [(d, d) for d in DTYPES] + [(torch.bfloat16, torch.float32)],
                         ids=str)
def test_steps_follow_the_formula_bit_for_bit(device, dtype, gdtype, master, bits, offset):
    """Three steps.  The kernel's operations are IEEE ones in a stated order, so fp32 on the
    CPU gives the same bits; the 64-bit formula is met to fp32 rounding."""
    params, grads = tensors(device, dtype, gdtype, offset=offset)
    opt = fm.AdamW(params, bits=bits, masters=master, **HYPER)
    work = [np32(p) for p in params]
    moments = [(np.zeros_like(w), np.zeros_like(w)) for w in work]
    for step in range(1, 4):
        opt.step([g * step for g in grads])
        got_m, got_v = opt.moment_values()
        for i, (w, g) in enumerate(zip(work, grads)):
            m, v = moments[i]
            g = np32(g * step)
            w64, m64, v64 = w.astype(float), m.astype(float), v.astype(float)
            p, m, v = step32(w, g, m, v, step, **HYPER)
            if bits == 8:
                codes = encode(m, True), encode(v, False)
                assert np.array_equal(opt.m[i].codes.cpu().numpy(), codes[0][0])
                assert np.array_equal(opt.v[i].codes.cpu().numpy(), codes[1][0])
                assert np.array_equal(opt.m[i].scales.cpu().numpy(), codes[0][1])
                m, v = decode(*codes[0]), decode(*codes[1])
            assert np.array_equal(np32(got_m[i]), m) and np.array_equal(np32(got_v[i]), v)
            moments[i] = m, v
            if master and dtype != torch.float32:
                assert np.array_equal(np32(opt.masters[i]), p)
            rounded = torch.from_numpy(p).to(dtype)
            assert torch.equal(params[i].cpu(), rounded)
            work[i] = p if master else rounded.float().numpy()
            # the formula in 64 bits
            b1, b2 = HYPER["betas"]
            m64 = b1 * m64 + (1 - b1) * g
            v64 = b2 * v64 + (1 - b2) * g.astype(float) ** 2
            p64 = w64 * (1 - HYPER["lr"] * HYPER["weight_decay"]) - HYPER["lr"] / (1 - b1 ** step) * (
                m64 / (np.sqrt(v64) / math.sqrt(1 - b2 ** step) + HYPER["eps"]))
            assert np.all(np.abs(p - p64) <= 2e-6 * (np.abs(w64) + 10 * HYPER["lr"]))


@pytest.mark.parametrize("count", [1, 150, 479, 480, 481, 1000])
def test_many_tensors(device, count):
    """Lists shorter and longer than a launch takes, empty tensors among them."""
    sizes = [(37 * i) % 900 for i in range(count)]
    params, grads = tensors(device, torch.float32, sizes=sizes)
    want = [step32(np32(p), np32(g), 0 * np32(p), 0 * np32(p), 1, **HYPER)[0]
            for p, g in zip(params, grads)]
    fm.AdamW(params, **HYPER).step(grads)
    assert all(np.array_equal(np32(p), w) for p, w in zip(params, want))


def test_eight_bit_codes_cover_their_range(device):
    """A block of magnitudes over twelve decades: a v above zero keeps a code, m's error is half a
    step of its code."""
    p = [torch.zeros(512, device=device)]
    g = [torch.logspace(-6, 0, 512, device=device)]
    opt = fm.AdamW(p, bits=8, **HYPER)
    opt.step(g)
    (m,), (v,) = opt.moment_values()
    assert (opt.v[0].codes > 0).all()
    true_m = 0.1 * g[0]
    a = opt.m[0].scales.repeat_interleave(256)
    root = (true_m / a).sqrt()
    assert ((m / a).sqrt() - root).abs().max() <= 0.5 / 127 + 1e-5
    true_v = 0.01 * g[0] ** 2
    root = (true_v / opt.v[0].scales.repeat_interleave(256)) ** 0.25
    got = (v / opt.v[0].scales.repeat_interleave(256)) ** 0.25
    assert (got - root).abs().max() <= 0.5 / 255 + 1e-5 or (root < 1 / 255).any()


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_and_non_finite_gradients(device, bits):
    """Zero gradients decay the weights and nothing else; a NaN or infinity shows in the element
    (32 bits) or its block (8 bits) and nowhere else."""
    p, g = [torch.ones(1000, device=device)], [torch.zeros(1000, device=device)]
    opt = fm.AdamW(p, bits=bits, **HYPER)
    opt.step(g)
    assert torch.equal(p[0], torch.full_like(p[0], np.float32(1 - HYPER["lr"] * HYPER["weight_decay"])))
    for bad in (math.nan, math.inf):
        p, g = tensors(device, torch.float32, sizes=[1000])
        clean = [p[0].clone()]
        fm.AdamW(clean, bits=bits, **HYPER).step(g)
        opt = fm.AdamW(p, bits=bits, **HYPER)
        dirty = g[0].clone()
        dirty[300] = bad
        opt.step([dirty])
        keep = torch.arange(1000, device=device) != 300
        assert torch.equal(p[0][keep], clean[0][keep]) and torch.isnan(p[0][300])
        opt.step(g)  # the block's moments are NaN now, the others are not
        block = (torch.arange(1000, device=device) // 256) == 1
        assert torch.isfinite(p[0][~block]).all()
        assert torch.isnan(p[0][block]).all() if bits == 8 else torch.isfinite(p[0][keep]).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_non_finite_moments_have_no_values(device, bad):
    """8-bit moments with a NaN or infinity among them are NaN throughout their block."""
    g = torch.sin(torch.arange(600, device=device) + 1.0)
    g[300] = bad
    opt = fm.AdamW([torch.ones(600, device=device)], bits=8, **HYPER)
    opt.step([g])
    block = torch.arange(600, device=device) // 256 == 1
    for (values,), moment in zip(opt.moment_values(), (opt.m[0], opt.v[0])):
        assert torch.isnan(values[block]).all() and torch.isfinite(values[~block]).all()
        assert torch.isnan(moment.scales).tolist() == [False, True, False]


def test_step_arguments(device):
    params, grads = tensors(device, torch.float32, sizes=[300, 20])
    before = [p.clone() for p in params]
    # a missing gradient leaves its tensor and moments as they are
    opt = fm.AdamW(params, **HYPER)
    opt.step([None, grads[1]])
    assert torch.equal(params[0], before[0]) and not opt.m[0].any() and opt.m[1].any()
    # grad_scale and lr of the call
    a, b = [before[0].clone()], [before[0].clone()]
    fm.AdamW(a, **HYPER).step([grads[0] * 0.5], lr=1e-2)
    fm.AdamW(b, **(HYPER | dict(lr=1e-2))).step([grads[0]], grad_scale=0.5)
    assert torch.equal(a[0], b[0])
    # going on from given moments is going on
    c, d = [before[0].clone()], [before[0].clone()]
    one = fm.AdamW(c, **HYPER)
    one.step([grads[0]])
    one.step([grads[0]])
    two = fm.AdamW(d, **HYPER)
    two.step([grads[0]])
    fm.AdamW(d, moments=(two.m, two.v), step=1, **HYPER).step([grads[0]])
    assert torch.equal(c[0], d[0])
    # the parameters' own gradients, and autograd notices that they moved
    w = before[0].clone().requires_grad_()
    y = (w * w).sum()
    y.backward(retain_graph=True)
    fm.AdamW([w], **HYPER).step()
    with pytest.raises(RuntimeError):
        y.backward()


def test_against_torch(device):
    """torch's own AdamW, ten steps: the same formula in another order of operations."""
    w = torch.randn(5000, device=device)
    a, b = w.clone().requires_grad_(), w.clone().requires_grad_()
    ours, theirs = fm.AdamW([a], **HYPER), torch.optim.AdamW([b], foreach=False, fused=False, **HYPER)
    for i in range(10):
        a.grad = torch.sin(w * (i + 1))
        b.grad = a.grad.clone()
        ours.step()
        theirs.step()
    torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


def test_other_stream_and_graph(device):
    params, grads = tensors(device, torch.bfloat16, sizes=[3000, 10])
    other = [p.clone() for p in params]
    fm.AdamW(params, bits=8, **HYPER).step(grads)
    side = torch.cuda.Stream(device)
    opt = fm.AdamW(other, bits=8, **HYPER)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        opt.step(grads)
    torch.cuda.current_stream(device).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(params, other))


def test_stepped_on_another_stream_and_dropped(device):
    """The memory of an optimiser that is dropped after a step on a stream of its own is not
    given out again before that step."""
    params, grads = tensors(device, torch.float32, sizes=[70001] * 4)
    other = [p.clone() for p in params]
    fm.AdamW(params, **HYPER).step(grads)
    moments = [[torch.zeros_like(p) for p in other] for _ in range(2)]
    opt = fm.AdamW(other, moments=moments, **HYPER)
    nbytes = opt._device_plan.numel()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    busy = torch.ones(4096, 4096, device=device)
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy @ busy * 2.0 ** -12
        opt.step(grads)
    at = opt._device_plan.data_ptr()
    del opt
    later = [torch.empty(nbytes, dtype=torch.uint8, device=device) for _ in range(8)]
    assert all(t.data_ptr() != at for t in later)
    torch.cuda.current_stream(device).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(params, other))


def test_refusals(device):
    p = [torch.zeros(8, device=device)]
    with pytest.raises(fm.ArgumentError):
        fm.AdamW(p, bits=4)
    with pytest.raises(fm.ArgumentError):
        fm.AdamW(p, betas=(1.0, 0.9))
    with pytest.raises(fm.ArgumentError):
        fm.AdamW([torch.zeros(8)])
    with pytest.raises(fm.UnsupportedError):
        fm.AdamW([p[0].double()])
    with pytest.raises(fm.DimensionMismatch):
        fm.AdamW(p, moments=([torch.zeros(7, device=device)], [torch.zeros(8, device=device)]))
    with pytest.raises(fm.ArgumentError):
        fm.AdamW(p, moments=([p[0].half()], [p[0]]))
    with pytest.raises(fm.ArgumentError):
        fm.AdamW(p, moments=([fm.Moment8.zeros(p[0], True)], [torch.zeros(8, device=device)]))
    with pytest.raises(fm.DimensionMismatch):
        fm.AdamW(p, masters=[torch.zeros(9, device=device)])
    opt = fm.AdamW(p)
    with pytest.raises(fm.DimensionMismatch):
        opt.step([])
    with pytest.raises(fm.DimensionMismatch):
        opt.step([torch.zeros(9, device=device)])
    with pytest.raises(fm.ArgumentError):
        opt.step([torch.zeros(16, device=device)[::2]])
    with pytest.raises(fm.ArgumentError):
        opt.step([torch.zeros(8)])
    p[0].data = torch.zeros(4, device=device)
    with pytest.raises(fm.DimensionMismatch):
        opt.step([torch.zeros(4, device=device)])
    with pytest.raises(fm.DimensionMismatch):
        fm.Moment8(torch.zeros(300, dtype=torch.int8), torch.zeros(1))
    with pytest.raises(fm.DimensionMismatch):
        fm.moment_values([fm.Moment8.zeros(torch.zeros(8, device=device), True)], [])
    assert opt.steps == 0


def test_arrays_lie_apart(device):
    """No array of a step may share memory with another; neighbours in one buffer may be stepped."""
    whole = torch.zeros(600, device=device)
    m, v = torch.zeros(300, device=device), torch.zeros(300, device=device)
    opt = fm.AdamW([whole[:300], whole[300:]], **HYPER)
    opt.step([torch.ones(300, device=device)] * 2)
    assert (whole == whole[0]).all() and whole[0] < 0
    for params, given in (([whole, whole[300:]], {}), ([whole[:301], whole[300:]], {}),
                          ([whole[:300], whole[:300].view(3, 100)], {}),
                          ([whole[:300]], dict(moments=([m], [m]))),
                          ([whole[:300]], dict(moments=([m], [v]), masters=[whole[:300]])),
                          ([whole[:300]], dict(moments=([m], [whole[200:500]])))):
        with pytest.raises(fm.ArgumentError, match="share memory"):
            fm.AdamW(params, **given)
    p = [torch.zeros(300, device=device), torch.zeros(300, device=device)]
    opt = fm.AdamW(p, **HYPER)
    p[0].data = p[1].data
    for _ in range(2):  # (refused once more, not stepped where it was)
        with pytest.raises(fm.ArgumentError, match="share memory"):
            opt.step([m, v])
    p[0].data = m
    opt.step([v, v])
    assert opt.steps == 1
    opt = fm.AdamW([torch.zeros(0, device=device), torch.zeros(0, device=device)], bits=8)
    opt.step([torch.zeros(0, device=device)] * 2)


def test_parameters_may_move(device):
    """A parameter given new memory is stepped there; one turned into a strided view is refused."""
    params, grads = tensors(device, torch.float32, sizes=[300, 64])
    other = [p.clone() for p in params]
    opt, ref = fm.AdamW(params, **HYPER), fm.AdamW(other, **HYPER)
    opt.step(grads)
    old = params[0].data
    params[0].data = params[0].data.clone()
    kept = old.clone()
    opt.step(grads)
    ref.step(grads)
    ref.step(grads)
    assert all(torch.equal(a, b) for a, b in zip(params, other)) and torch.equal(old, kept)
    params[1].data = params[1].data.view(8, 8).t()
    with pytest.raises(fm.ArgumentError):
        opt.step(grads)
