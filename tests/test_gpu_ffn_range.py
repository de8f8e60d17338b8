"""What the gated feed-forward's pullback keeps of dg and du, the cotangents of the projections,
on their way into the products that sum them: as much as fp32 does, at any size of the cotangent.

The outputs are rounded once, so the bound is the error of the 64-bit result's own rounding to the
type, in the 2-norm, times 1.1.  What may be added to it: 2^-17 of dg and du for holding them
(16-bit types), against the rounding's 2^-9 or 2^-12, and fp32 sums of some thousand terms, 2^-24
sqrt(terms) = 2^-18; both together change the norm by less than 2 %.  One rounding of dg and du to
the type would multiply it by 1.4, the loss of their range by far more.
"""
import math

import pytest
import torch

import flashmaxsim as fm
from test_gpu_ffn import act64

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


def make(device, t, k, f, dtype, dh=0.1, x=1.0, wg=1.0, wu=1.0, seed=0):
    """Inputs of the given scales; dh may be a scale for each token."""
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(rows, cols, scale):
        return (torch.randn(rows, cols, generator=g, device=device) * scale).to(dtype)

    s = k ** -0.5
    return normal(t, k, x), normal(f, k, wg * s), normal(f, k, wu * s), normal(t, f, dh)


def exact(x, wg, wu, dh, act):
    x, wg, wu, dh = (a.double() for a in (x, wg, wu, dh))
    g, u = x @ wg.T, x @ wu.T
    a, da = act64(g, act)
    dg, du = dh * u * da, dh * a
    return (dg @ wg + du @ wu, dg.T @ x, du.T @ x), dg


def check(got, want, dtype, what, rows=None):
    """rows: compare each row by itself (rows of very different sizes)."""
    off, own = got.double() - want, want.to(dtype).double() - want
    dims = (0, 1) if rows is None else 1
    assert torch.isfinite(got).all(), what
    off, own = off.pow(2).sum(dims).sqrt(), own.pow(2).sum(dims).sqrt()
    assert (off <= 1.1 * own).all(), (what, float((off / own).max()))


def run(inputs, act, dtype, what, rows=None):
    want, dg = exact(*inputs, act)
    x, wg, wu, dh = inputs
    for name, got, w in zip(("dx", "dwg", "dwu"), fm.gated_ffn_pullback(dh, x, wg, wu, act), want):
        check(got, w, dtype, (what, name), rows if name == "dx" else None)
    return dg


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("size", [1e-6, 1e-5, 0.1, 10.0])
@pytest.mark.parametrize("dtype", HALVES, ids=str)
def test_small_and_ordinary_cotangents(device, dtype, size, act):
    """8192 tokens: sums over them would hide nothing of what each term lost."""
    run(make(device, 8192, 128, 128, dtype, dh=size), act, dtype, size)


@pytest.mark.parametrize("dtype", HALVES, ids=str)
@pytest.mark.parametrize("shape", [(6200, 264, 1032), (1237, 200, 531), (300, 40, 1000), (9, 24, 17)], ids=str)
def test_every_shape_of_tile(device, shape, dtype):
    """Large tiles, small ones, rows that are no whole 16-byte units, long sums cut into parts."""
    run(make(device, *shape, dtype, dh=1e-3), "silu", dtype, shape)


def test_values_past_the_type_inside(device):
    """fp16: dg reaches infinity as fp16 although no output does."""
    inputs = make(device, 4, 64, 64, torch.float16, dh=1e4, x=0.01, wg=8e-3, wu=4e3)
    dg = run(inputs, "silu", torch.float16, "large")
    assert dg.abs().max() > 65504


@pytest.mark.parametrize("dtype,sizes", [(torch.float16, (30.0, 1.0, 1e-3, 1e-5)),
                                         (torch.bfloat16, (1e10, 1.0, 1e-12, 1e-25))], ids=str)
def test_tokens_of_different_sizes(device, dtype, sizes):
    """Each token's dx is as good as if it were alone."""
    scale = torch.tensor(sizes, device=device).repeat(64)[:, None]
    run(make(device, 256, 64, 64, dtype, dh=scale), "silu", dtype, sizes, rows=True)


@pytest.mark.parametrize("dtype", HALVES, ids=str)
def test_zero_cotangents(device, dtype):
    x, wg, wu, dh = make(device, 200, 64, 72, dtype)
    for a, b in ((dh * 0, x), (dh, x * 0)):
        dx, dwg, dwu = fm.gated_ffn_pullback(a, b, wg, wu)
        assert not dx.any() and not dwg.any() and not dwu.any()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", HALVES, ids=str)
def test_what_is_not_finite_stays_where_it_was(device, dtype, bad):
    """A token that is not finite shows in its dx alone, a cotangent that is not also in its hidden
    unit's weights; the rest is as exact as without it."""
    x, wg, wu, dh = make(device, 300, 72, 136, dtype, dh=1e-5)
    keep, hidden = torch.arange(300, device=device) != 1, torch.arange(136, device=device) != 7
    y = x.clone()
    y[1] = bad
    got = fm.gated_ffn_pullback(dh, y, wg, wu)[0]
    check(got[keep], exact(x[keep], wg, wu, dh[keep], "silu")[0][0], dtype, "dx")
    assert not torch.isfinite(got[1]).any()
    d = dh.clone()
    d[1, 7] = bad
    dx, dwg, dwu = fm.gated_ffn_pullback(d, x, wg, wu)
    want = exact(x, wg, wu, dh, "silu")[0]
    check(dx[keep], want[0][keep], dtype, "dx")
    check(dwg[hidden], want[1][hidden], dtype, "dwg")
    check(dwu[hidden], want[2][hidden], dtype, "dwu")
    assert not torch.isfinite(dx[1]).any()
    assert not torch.isfinite(dwg[7]).any() and not torch.isfinite(dwu[7]).any()


@pytest.mark.parametrize("shape", [(500, 100, 60), (300, 64, 136)], ids=str)
def test_replayed_with_other_sizes(device, shape):
    """A captured fp16 pullback finds the range of what it is replayed on."""
    x, wg, wu, dh = make(device, *shape, torch.float16, dh=1.0)
    d = dh.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fm.gated_ffn_pullback(d, x, wg, wu)
    for scale in (1.0, 1e-5, 30.0, 0.0):
        d.copy_(dh * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, fm.gated_ffn_pullback(d, x, wg, wu)))
        for got, want in zip(out, exact(x, wg, wu, d, "silu")[0]):
            check(got, want, torch.float16, scale)
