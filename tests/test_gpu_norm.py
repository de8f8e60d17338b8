"""The block norms on the GPU against their formula in 64 bits, gradients by differentiating it.

Bounds: fp32 arithmetic on a row (2^-24 for each operation of a sum over dim), one rounding
of each output to the feature type.
"""
import itertools

import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FORMS = {"pre": (False, False, True), "post": (True, True, False), "plain": (True, False, True),
         "both": (True, True, True), "add": (True, False, False)}


def make(device, lead, dim, dtype, form, gate, seed=0, offset=0):
    g = torch.Generator().manual_seed(seed + dim)
    has_f, has_post, has_pre = FORMS[form]

    def normal(*shape, scale=1.0, shift=0.0):
        n = torch.Size(shape).numel()
        x = torch.empty(n + offset, dtype=dtype)
        x[offset:] = (torch.randn(n, generator=g) * scale + shift).to(dtype)
        return x.to(device)[offset:].view(*shape)

    a = {"x": normal(*lead, dim, scale=1.5), "f": normal(*lead, dim, shift=0.2) if has_f else None,
         "gate": None, "post_weight": normal(dim, scale=0.1, shift=1.0) if has_post else None,
         "pre_weight": normal(dim, scale=0.1, shift=1.0) if has_pre else None}
    if has_f and gate is not None:
        a["gate"] = normal(*lead[:gate], dim, scale=0.3, shift=0.5)
    a["dr"] = normal(*lead, dim, scale=0.1)
    a["dn"] = normal(*lead, dim, scale=0.1) if has_pre else None
    return a


def reference(a, scale, kind, eps):
    names = [k for k in ("x", "f", "gate", "post_weight", "pre_weight") if a[k] is not None]
    v = {k: a[k].detach().cpu().double().requires_grad_() for k in names}

    def norm(t, w):
        if kind == "layer":
            t = t - t.mean(-1, keepdim=True)
        return t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps) * w

    r = v["x"]
    if "f" in v:
        z = norm(v["f"], v["post_weight"]) if "post_weight" in v else v["f"]
        if "gate" in v:
            gate = v["gate"]
            z = z * gate.reshape(gate.shape[:-1] + (1,) * (z.dim() - gate.dim()) + gate.shape[-1:])
        r = r + scale * z
    n = norm(r, v["pre_weight"]) if "pre_weight" in v else None
    total = (r * a["dr"].cpu().double()).sum()
    if n is not None:
        total = total + (n * a["dn"].cpu().double()).sum()
    grads = dict(zip(names, torch.autograd.grad(total, list(v.values()))))
    return r.detach(), None if n is None else n.detach(), grads


def close(got, want, dtype, terms, what):
    """Within one rounding to the type and `terms` fp32 roundings of the tensor's scale."""
    got, want = got.detach().cpu().double(), want
    assert got.shape == want.shape, what
    scale = float(want.pow(2).mean().sqrt()) if want.numel() else 0.0
    bound = 1.02 * HALF_ULP[dtype] * want.abs() + terms * 2.0 ** -24 * (want.abs() + scale) + 1e-7
    off = (got - want).abs()
    assert (off <= bound).all(), (what, float((off / bound).max()))


def run(device, lead, dim, dtype, form, gate, kind, offset=0, eps=1e-6):
    a = make(device, lead, dim, dtype, form, gate, offset=offset)
    args = {k: a[k] for k in ("gate", "post_weight", "pre_weight")} | dict(scale=0.7, kind=kind, eps=eps)
    r, n = fm.block_norm_forward(a["x"], a["f"], **args)
    grads = fm.block_norm_pullback(a["dr"], a["dn"], a["x"], a["f"], **args)
    wr, wn, wg = reference(a, 0.7, kind, eps)
    rows = max(1, torch.Size(lead).numel())
    close(r, wr, dtype, 8 + dim ** 0.5, "r")
    if wn is not None:
        close(n, wn, dtype, 16 + 2 * dim ** 0.5, "n")
    for name, got in zip(("x", "f", "gate", "post_weight", "pre_weight"), grads):
        assert (got is None) == (name not in wg), name
        if got is not None:
            close(got, wg[name], dtype, 64 + 4 * dim ** 0.5 + 4 * rows ** 0.5, "d" + name)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("form,gate", [("pre", None)] + list(itertools.product(
    ("post", "plain", "both", "add"), (None, 0, 1, 2))), ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_forms(device, dtype, form, gate, kind):
    """Every form with every gate: none, shared, one a sequence, one a token."""
    run(device, (5, 7), 72, dtype, form, gate, kind)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim", [2, 3, 64, 65, 511, 512, 513, 1000, 1024, 1025, 1537, 2048, 2056, 4096,
                                 4100, 9000, 16384])
def test_widths(device, dim, dtype):
    run(device, (3, 4), dim, dtype, "both", 1, "layer")


@pytest.mark.parametrize("lead,gate", [((1,), 0), ((1, 1), 1), ((700,), 0), ((2, 1500), 1),
                                       ((900, 3), 1), ((300, 2, 2), 1), ((13, 333), 0)], ids=str)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_and_gate_groups(device, lead, gate, kind):
    """Column sums over one row, many rows, groups that workgroups share or split."""
    run(device, lead, 96, torch.float32, "both", gate, kind)


@pytest.mark.parametrize("offset", [1, 3])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_bases_off_16_bytes(device, dtype, offset):
    run(device, (4, 5), 128, dtype, "both", 1, "rms", offset=offset)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_of_zeros(device, kind):
    """A padding row: its norm is zero and its gradient finite, 1 / sqrt(eps) times the cotangent."""
    x = torch.zeros(3, 64, device=device)
    x[1] = torch.randn(64, device=device)
    w = torch.ones(64, device=device)
    _, n = fm.block_norm_forward(x, pre_weight=w, kind=kind, eps=1e-4)
    assert not n[0].any() and not n[2].any() and n[1].any()
    dn = torch.randn(3, 64, device=device)
    dx = fm.block_norm_pullback(None, dn, x, pre_weight=w, kind=kind, eps=1e-4)[0]
    want = dn[0] - (dn[0].mean() if kind == "layer" else 0)
    torch.testing.assert_close(dx[0], want * 100, rtol=1e-5, atol=1e-4)


def test_nan_and_infinity_stay_in_their_row(device):
    x = torch.randn(9, 200, device=device)
    w = torch.ones(200, device=device)
    f = torch.randn_like(x)
    clean = fm.block_norm_forward(x, f, post_weight=w, pre_weight=w)
    y, g = x.clone(), f.clone()
    y[2, 5], g[6, 100] = float("inf"), float("nan")
    got = fm.block_norm_forward(y, g, post_weight=w, pre_weight=w)
    keep = torch.tensor([i not in (2, 6) for i in range(9)], device=device)
    for a, b in zip(got, clean):
        assert torch.equal(a[keep], b[keep])
        assert torch.isnan(got[1][2]).any() and torch.isnan(got[1][6]).all()


@pytest.mark.parametrize("shape", [(0, 8), (4, 0), (0, 3, 8)], ids=str)
def test_empty(device, shape):
    x = torch.zeros(shape, device=device)
    w = torch.ones(shape[-1], device=device)
    r, n = fm.block_norm_forward(x, x, gate=w, post_weight=w, pre_weight=w)
    assert r.shape == n.shape == x.shape
    grads = fm.block_norm_pullback(x, x, x, x, gate=w, post_weight=w, pre_weight=w)
    assert [g.shape for g in grads] == [x.shape, x.shape, w.shape, w.shape, w.shape]
    assert not any(g.any() for g in grads)


def test_cotangents_may_be_missing(device):
    a = make(device, (6,), 64, torch.float32, "both", 0)
    args = {k: a[k] for k in ("gate", "post_weight", "pre_weight")}
    zero = torch.zeros_like(a["x"])
    for dr, dn in ((a["dr"], None), (None, a["dn"]), (None, None)):
        got = fm.block_norm_pullback(dr, dn, a["x"], a["f"], **args)
        want = fm.block_norm_pullback(zero if dr is None else dr, zero if dn is None else dn, a["x"],
                                      a["f"], **args)
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_autograd_and_repeats(device):
    a = make(device, (4, 50), 256, torch.float32, "both", 1)
    names = ("x", "f", "gate", "post_weight", "pre_weight")
    want = fm.block_norm_pullback(a["dr"], a["dn"], a["x"], a["f"], **{k: a[k] for k in names[2:]})
    leaves = {k: a[k].clone().requires_grad_() for k in names}
    r, n = fm.block_norm(leaves["x"], leaves["f"], **{k: leaves[k] for k in names[2:]})
    torch.autograd.backward([r, n], [a["dr"], a["dn"]])
    assert all(torch.equal(leaves[k].grad, w) for k, w in zip(names, want))
    x = a["x"].clone().requires_grad_()
    r, n = fm.block_norm(x, pre_weight=a["pre_weight"])
    assert r is x
    n.sum().backward()
    assert torch.equal(x.grad, fm.block_norm_pullback(None, torch.ones_like(n), a["x"],
                                                      pre_weight=a["pre_weight"])[0])
    for _ in range(2):
        again = fm.block_norm_pullback(a["dr"], a["dn"], a["x"], a["f"], **{k: a[k] for k in names[2:]})
        assert all(torch.equal(g, w) for g, w in zip(again, want))


def test_gradient_against_differences(device):
    """Central differences in fp32, steps of 1e-2 of a value: truncation and rounding of 1e-3."""
    a = make(device, (3, 8), 40, torch.float32, "both", 1)
    names = ("x", "f", "gate", "post_weight", "pre_weight")
    for kind in ("rms", "layer"):
        grads = fm.block_norm_pullback(a["dr"], a["dn"], a["x"], a["f"], kind=kind,
                                       **{k: a[k] for k in names[2:]})

        def loss(b):
            r, n = fm.block_norm_forward(b["x"], b["f"], kind=kind, **{k: b[k] for k in names[2:]})
            return float((r.double() * a["dr"].double()).sum() + (n.double() * a["dn"].double()).sum())

        for name, grad in zip(names, grads):
            v = torch.randn_like(a[name])
            ends = [loss(a | {name: a[name] + s * v}) for s in (5e-3, -5e-3)]
            want = (ends[0] - ends[1]) / 1e-2
            got = float((grad.double() * v.double()).sum())
            assert abs(got - want) <= 5e-3 * float(grad.double().norm() * v.double().norm()), (kind, name)


def test_other_stream_and_graph(device):
    a = make(device, (40, 30), 200, torch.bfloat16, "both", 1)
    args = {k: a[k] for k in ("gate", "post_weight", "pre_weight")}

    def both(x):
        return (fm.block_norm_forward(x, a["f"], **args)
                + fm.block_norm_pullback(a["dr"], a["dn"], x, a["f"], **args))

    want = both(a["x"])
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        got = both(a["x"])
    torch.cuda.current_stream(device).wait_stream(side)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    x = a["x"].clone()
    with torch.cuda.graph(graph):
        out = both(x)
    for i in range(3):
        x.copy_(a["x"] * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(out, both(x)))


def test_refusals(device):
    x, w = torch.ones(4, 8, device=device), torch.ones(8, device=device)
    with pytest.raises(fm.ArgumentError):
        fm.block_norm_forward(x)  # nothing to compute
    with pytest.raises(fm.ArgumentError):
        fm.block_norm_forward(x, gate=w, pre_weight=w)  # a gate without a branch
    with pytest.raises(fm.ArgumentError):
        fm.block_norm_forward(x, pre_weight=w, kind="batch")
    with pytest.raises(fm.ArgumentError):
        fm.block_norm_forward(x, pre_weight=w.half())
    with pytest.raises(fm.ArgumentError):
        fm.block_norm_forward(x.cpu(), pre_weight=w)
    with pytest.raises(fm.ArgumentError):
        fm.block_norm_pullback(None, x, x, x)  # dn without pre_weight
    with pytest.raises(fm.DimensionMismatch):
        fm.block_norm_forward(x, x[:3], pre_weight=w)
    with pytest.raises(fm.DimensionMismatch):
        fm.block_norm_forward(x, x, gate=x[:2])
    with pytest.raises(fm.DimensionMismatch):
        fm.block_norm_forward(x, pre_weight=w[:4])
    big = torch.ones(1, 16385, device=device)
    with pytest.raises(fm.UnsupportedError):
        fm.block_norm_forward(big, pre_weight=big[0])
