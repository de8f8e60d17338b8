"""The gated feed-forward block on the GPU against its formula in 64 bits.

Every bound is the rounding the formula allows, element by element: fp32 products summed
in any order (2^-24 of the sum of magnitudes for each term), the activation's few units in the
last place, one rounding of each output to the feature type, and one of dg and du between the
pullback's products.
"""
import math

import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 1e-37, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-37}
F32 = 2.0 ** -24
SHAPES = [(1, 1, 1), (1, 8, 16), (3, 7, 5), (2, 128, 64), (16, 64, 48), (17, 96, 33), (33, 64, 40),
          (64, 256, 130), (65, 200, 77), (130, 129, 257), (257, 72, 300), (5, 1000, 8),
          (300, 40, 1000)]


def act64(g, act):
    """act(g), act'(g) in 64 bits."""
    g = g.clone().requires_grad_()
    if act == "silu":
        a = g * torch.sigmoid(g)
    elif act == "gelu":
        a = 0.5 * g * torch.special.erfc(-g / math.sqrt(2))
    else:
        a = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    return a.detach(), torch.autograd.grad(a.sum(), g)[0]


def inputs(device, t, k, f, dtype, seed=0, offset=0):
    g = torch.Generator().manual_seed(seed + 1000 * t + 100 * k + f)

    def make(*shape, scale):
        n = math.prod(shape)
        x = torch.empty(n + offset, dtype=dtype)
        x[offset:] = (torch.randn(n, generator=g) * scale).to(dtype)
        return x.to(device)[offset:].view(*shape)

    s = max(k, 1) ** -0.5
    return make(t, k, scale=1.0), make(f, k, scale=s), make(f, k, scale=s), make(t, f, scale=0.1)


def reference(x, wg, wu, dh, act, dtype, where="cpu"):
    """{name: (value, bound)} in 64 bits."""
    u_out, least = HALF_ULP[dtype], LEAST[dtype]
    x, wg, wu, dh = (a.to(where).double() for a in (x, wg, wu, dh))
    k, f, t = x.shape[1], wg.shape[0], x.shape[0]
    g, u = x @ wg.T, x @ wu.T
    eg = 2 * F32 * (k + 2) * (x.abs() @ wg.abs().T)
    eu = 2 * F32 * (k + 2) * (x.abs() @ wu.abs().T)
    a, da = act64(g, act)
    # |act'| <= 1.2 and |act''| <= 1; the functions themselves to 16 units at 1 + |g|
    ea = 1.2 * eg + 16 * F32 * (1 + g.abs())
    eda = eg + 16 * F32 * (1 + g.abs())
    out = {}

    def rounded(v, e):
        return v, e + (1.01 * u_out if dtype != torch.float32 else 2 * F32) * (v.abs() + e) + least

    out["h"] = rounded(a * u, ea * (u.abs() + eu) + a.abs() * eu)
    dg, edg = rounded(dh * u * da, dh.abs() * ((u.abs() + eu) * eda + eu * da.abs()))
    du, edu = rounded(dh * a, dh.abs() * ea)
    edx = edg @ wg.abs() + edu @ wu.abs()
    adx = (dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()
    out["dx"] = rounded(dg @ wg + du @ wu, edx + 2 * F32 * (2 * f + 2) * adx)
    for name, d, ed in (("dwg", dg, edg), ("dwu", du, edu)):
        out[name] = rounded(d.T @ x, ed.T @ x.abs() + 2 * F32 * (t + 2) * ((d.abs() + ed).T @ x.abs()))
    return out


def check(got, want, what):
    value, bound = want
    off = (got.to(value.device).double() - value).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), bad.numel(), float((off / bound).max()))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_pullback(device, shape, dtype, act):
    x, wg, wu, dh = inputs(device, *shape, dtype)
    want = reference(x, wg, wu, dh, act, dtype)
    check(fm.gated_ffn_forward(x, wg, wu, act), want["h"], "h")
    for name, got in zip(("dx", "dwg", "dwu"), fm.gated_ffn_pullback(dh, x, wg, wu, act)):
        check(got, want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1500, 264, 520), (40, 512, 2048), (4200, 64, 48), (700, 1032, 136),
                                   (6200, 264, 1032)], ids=str)
def test_many_tiles(device, shape, dtype):
    """Several tiles each way, the large tile among them, and long sums cut into parts."""
    x, wg, wu, dh = inputs(device, *shape, dtype)
    want = reference(x, wg, wu, dh, "silu", dtype)
    check(fm.gated_ffn_forward(x, wg, wu), want["h"], "h")
    for name, got in zip(("dx", "dwg", "dwu"), fm.gated_ffn_pullback(dh, x, wg, wu)):
        check(got, want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(6200, 264, 1037), (6200, 201, 1032), (9001, 513, 2055),
                                   (20011, 1000, 2000)], ids=str)
def test_large_and_odd(device, shape, dtype):
    """The large tiles with rows and widths that end inside them, whole 16-byte units or not."""
    x, wg, wu, dh = inputs(device, *shape, dtype)
    want = reference(x, wg, wu, dh, "gelu_tanh", dtype, device)
    check(fm.gated_ffn_forward(x, wg, wu, "gelu_tanh"), want["h"], "h")
    for name, got in zip(("dx", "dwg", "dwu"), fm.gated_ffn_pullback(dh, x, wg, wu, "gelu_tanh")):
        check(got, want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens, dim", [(1, 520), (16, 16), (17, 1029), (33, 520), (48, 1024), (64, 513),
                                         (65, 520), (200, 72)])
@pytest.mark.parametrize("hidden", [3, 2048, 2049])
def test_few_tokens(device, tokens, dim, hidden, dtype):
    """Few tokens, on both sides of where their kernel changes its share of hidden units."""
    x, wg, wu, dh = inputs(device, tokens, dim, hidden, dtype)
    want = reference(x, wg, wu, dh, "silu", dtype, device)
    check(fm.gated_ffn_forward(x, wg, wu), want["h"], "h")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_bases_off_16_bytes(device, dtype, offset):
    x, wg, wu, dh = inputs(device, 70, 64, 72, dtype, offset=offset)
    want = reference(x, wg, wu, dh, "silu", dtype)
    check(fm.gated_ffn_forward(x, wg, wu), want["h"], "h")
    for name, got in zip(("dx", "dwg", "dwu"), fm.gated_ffn_pullback(dh, x, wg, wu)):
        check(got, want[name], name)


@pytest.mark.parametrize("shape", [(0, 8, 8), (4, 0, 8), (4, 8, 0), (0, 0, 0)], ids=str)
def test_empty(device, shape):
    t, k, f = shape
    x, wg, wu, dh = inputs(device, t, k, f, torch.bfloat16)
    h = fm.gated_ffn_forward(x, wg, wu)
    assert h.shape == (t, f) and not h.any()
    dx, dwg, dwu = fm.gated_ffn_pullback(dh, x, wg, wu)
    for d, like in ((dx, x), (dwg, wg), (dwu, wu)):
        assert d.shape == like.shape and not d.any()


def test_leading_dimensions_and_stacked_weights(device):
    x, wg, wu, _ = inputs(device, 12, 64, 40, torch.float16)
    w = torch.cat([wg, wu])
    a = fm.gated_ffn_forward(x.view(3, 4, 64), w[:40], w[40:])
    assert a.shape == (3, 4, 40)
    assert torch.equal(a.view(12, 40), fm.gated_ffn_forward(x, wg, wu))
    assert fm.gated_ffn_forward(x[0], wg, wu).shape == (40,)


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_a_row_of_nan_or_infinity_stays_in_its_row(device, tokens):
    x, wg, wu, dh = inputs(device, tokens, 72, 136, torch.bfloat16)
    clean = fm.gated_ffn_forward(x, wg, wu)
    cdx = fm.gated_ffn_pullback(dh, x, wg, wu, need_dw=False)[0]
    for bad in (math.nan, math.inf):
        y = x.clone()
        y[1] = bad
        h = fm.gated_ffn_forward(y, wg, wu)
        dx = fm.gated_ffn_pullback(dh, y, wg, wu, need_dw=False)[0]
        keep = torch.arange(tokens, device=device) != 1
        assert torch.equal(h[keep], clean[keep]) and torch.equal(dx[keep], cdx[keep])
        assert not torch.isfinite(h[1]).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_far_arguments(device, act):
    """Where the activation saturates: large positive passes, large negative vanishes, no NaN."""
    g = torch.tensor([-3e4, -300.0, -90.0, -20.0, -0.0, 0.0, 20.0, 90.0, 300.0, 3e4], device=device)
    one = torch.ones(1, 1, device=device)
    h = fm.gated_ffn_forward(g[:, None], one, one, act)[:, 0]
    a, da = act64(g.cpu().double(), act)
    torch.testing.assert_close(h.cpu().double(), a * g.cpu().double(), rtol=2e-6, atol=1e-6)
    dx = fm.gated_ffn_pullback(torch.ones_like(g)[:, None], g[:, None], one, one, act)[0][:, 0]
    want = (a + da * g.cpu().double())
    torch.testing.assert_close(dx.cpu().double(), want, rtol=2e-6, atol=1e-5)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_runs_repeat_bit_for_bit(device, dtype):
    x, wg, wu, dh = inputs(device, 3000, 128, 200, dtype)
    first = (fm.gated_ffn_forward(x, wg, wu),) + fm.gated_ffn_pullback(dh, x, wg, wu)
    for _ in range(3):
        again = (fm.gated_ffn_forward(x, wg, wu),) + fm.gated_ffn_pullback(dh, x, wg, wu)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_gradient_against_differences(device):
    """Central differences of the fp32 forward in random directions: the truncation is 1e-6 of
    the scale, the forward's rounding over the step 1e-4."""
    x, wg, wu, dh = inputs(device, 20, 24, 36, torch.float32)
    for act in ("silu", "gelu", "gelu_tanh"):
        grads = fm.gated_ffn_pullback(dh, x, wg, wu, act)
        for i in range(3):
            args = [x, wg, wu]
            v = torch.randn_like(args[i])
            step = 1e-2 / float(v.abs().max())
            ends = []
            for s in (step, -step):
                moved = list(args)
                moved[i] = args[i] + s * v
                ends.append((fm.gated_ffn_forward(*moved, act).double() * dh.double()).sum())
            want = float(ends[0] - ends[1]) / (2 * step)
            got = float((grads[i].double() * v.double()).sum())
            scale = float(grads[i].double().norm() * v.double().norm())
            assert abs(got - want) <= 2e-3 * scale, (act, i, got, want)


def test_autograd(device):
    x, wg, wu, dh = inputs(device, 10, 64, 48, torch.float32)
    want = fm.gated_ffn_pullback(dh, x, wg, wu)
    leaves = [a.clone().requires_grad_() for a in (x, wg, wu)]
    h = fm.gated_ffn(*leaves)
    h.backward(dh)
    assert all(torch.equal(a.grad, b) for a, b in zip(leaves, want))
    # a broadcast cotangent, and a weight that needs none
    xs = x.clone().requires_grad_()
    fm.gated_ffn(xs, wg, wu).sum().backward()
    assert torch.equal(xs.grad, fm.gated_ffn_pullback(torch.ones_like(dh), x, wg, wu)[0])


def test_other_stream_and_graph(device):
    x, wg, wu, dh = inputs(device, 500, 100, 60, torch.bfloat16)  # rows of 200 bytes: copied
    want = (fm.gated_ffn_forward(x, wg, wu),) + fm.gated_ffn_pullback(dh, x, wg, wu)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        got = (fm.gated_ffn_forward(x, wg, wu),) + fm.gated_ffn_pullback(dh, x, wg, wu)
    torch.cuda.current_stream(device).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    y = x.clone()
    with torch.cuda.graph(graph):
        out = (fm.gated_ffn_forward(y, wg, wu),) + fm.gated_ffn_pullback(dh, y, wg, wu)
    for i in range(3):
        y.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = (fm.gated_ffn_forward(y, wg, wu),) + fm.gated_ffn_pullback(dh, y, wg, wu)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_offsets_past_32_bits(device):
    """More than 2^32 bytes of h, dg and du: the last tokens come out as they do alone."""
    t, k, f = 600_000, 16, 4096
    g = torch.Generator(device=device).manual_seed(3)
    x = torch.randn(t, k, generator=g, device=device).to(torch.bfloat16)
    wg = torch.randn(f, k, generator=g, device=device).to(torch.bfloat16)
    h = fm.gated_ffn_forward(x, wg, wg)
    tail = slice(t - 256, t)
    assert torch.equal(h[tail], fm.gated_ffn_forward(x[tail], wg, wg))
    dx = fm.gated_ffn_pullback(h, x, wg, wg, need_dw=False)[0]
    want = reference(x[tail], wg, wg, h[tail], "silu", torch.bfloat16)["dx"]
    check(dx[tail], want, "dx")


def test_refusals(device):
    x, wg, wu, dh = inputs(device, 4, 8, 6, torch.float16)
    with pytest.raises(fm.ArgumentError):
        fm.gated_ffn_forward(x, wg, wu, "relu")
    with pytest.raises(fm.ArgumentError):
        fm.gated_ffn_forward(x.cpu(), wg, wu)
    with pytest.raises(fm.ArgumentError):
        fm.gated_ffn_forward(x, wg.float(), wu)
    with pytest.raises(fm.ArgumentError):
        fm.gated_ffn_forward(x.t().contiguous().t(), wg, wu)  # not dense
    with pytest.raises(fm.UnsupportedError):
        fm.gated_ffn_forward(x.double(), wg.double(), wu.double())
    with pytest.raises(fm.DimensionMismatch):
        fm.gated_ffn_forward(x, wg[:5].contiguous(), wu)
    with pytest.raises(fm.DimensionMismatch):
        fm.gated_ffn_forward(x[:, :4].contiguous(), wg, wu)
    with pytest.raises(fm.DimensionMismatch):
        fm.gated_ffn_pullback(dh[:3], x, wg, wu)
