"""The norm and rotation of heads and their pullback against the definition in 64 bits, every entry held to what
fp32 sums over a head (or over all tokens, for the weights) and one rounding may cost."""
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = 2.0 ** -24
EPS = 1e-6


def swap(x, turned, pairing):
    """The values as (a, b, rest): first and second values of the pairs, and what is not turned."""
    head, rest = x[..., :turned], x[..., turned:]
    if pairing == "halves":
        return head[..., :turned // 2], head[..., turned // 2:], rest
    return head[..., 0::2], head[..., 1::2], rest


def joined(a, b, rest, pairing):
    head = torch.cat([a, b], -1) if pairing == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([head, rest], -1)


def turn(x, cos, sin, turned, pairing):
    a, b, rest = swap(x, turned, pairing)
    return joined(a * cos - b * sin, b * cos + a * sin, rest, pairing)


def turn_size(x, turned, pairing):
    """What a turned entry's terms add up to at most."""
    a, b, rest = swap(x.abs(), turned, pairing)
    return joined(a + b, a + b, rest, pairing)


def reference(x, w, rows, turned, kind, pairing, dy, inside):
    """{name: (value, bound)} of one of the two, rows (..., 1, turned) the table's."""
    half = torch.finfo(x.dtype).eps / 2 * 1.001
    floor = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    d = x.shape[-1]
    u = UNIT * (d + 20)
    cos, sin = rows[..., :turned // 2].double(), rows[..., turned // 2:].double()
    x, dy, inside = x.double(), dy.double(), inside[..., None, None]
    y, xhat, size, inv = x, None, x.abs(), None
    if w is not None:
        centred = x - x.mean(-1, keepdim=True) if kind == "layer" else x
        inv = (centred.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        xhat = centred * inv
        # (the mean's own rounding is one of the whole head's size)
        hat_size = xhat.abs() + inv * x.abs().amax(-1, keepdim=True)
        # inv is off by half the relative error of the spread, to which a wrong mean adds
        hat_off = u * hat_size * (1 + (inv * x.abs().amax(-1, keepdim=True) if kind == "layer" else 0))
        y, size = xhat * w.double(), (hat_off / u) * w.double().abs()
    out = turn(y, cos, sin, turned, pairing)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    res = {"y": (torch.where(inside, out, zero), half * out.abs() + u * turn_size(size, turned, pairing) + floor)}
    g = torch.where(inside, turn(dy, cos, -sin, turned, pairing), zero)
    g_size = turn_size(dy, turned, pairing)
    if w is None:
        res["dx"] = (g, half * g.abs() + u * g_size + floor)
        return res
    lead = tuple(range(x.dim() - 1))
    count = x[..., 0].numel()
    dw = torch.where(inside, g * xhat, zero).sum(lead)
    dw_size = torch.where(inside, g_size * hat_off / u, zero).sum(lead)
    res["dw"] = (dw, half * dw.abs() + (u + count * UNIT) * dw_size + floor)
    gw = g * w.double()
    gw_size = g_size * w.double().abs()
    dx = gw - xhat * (gw * xhat).mean(-1, keepdim=True)
    dx = (dx - gw.mean(-1, keepdim=True) if kind == "layer" else dx) * inv
    hs = hat_off / u
    dx_size = (gw_size + hs * (gw_size * hs).mean(-1, keepdim=True) + gw_size.mean(-1, keepdim=True)) * inv
    spread = 1 + inv * x.abs().amax(-1, keepdim=True) if kind == "layer" else 1
    res["dx"] = (torch.where(inside, dx, zero), half * dx.abs() + 3 * u * dx_size * spread + floor)
    return res


def close(got, want, what):
    x, far = want
    assert got.shape == x.shape, (what, got.shape, x.shape)
    over = (got.double() - x).abs() / far
    assert torch.isfinite(got).all() and (not got.numel() or float(over.max()) <= 1.0), \
        f"{what}: {float(over.max()):.3f} times as far off as roundings may be"


def check(shape, kv_heads, turned, dtype, device, kind="rms", pairing="halves", weights="qk", positions=None,
          rows=None, view=None, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    *lead, tokens, heads, d = shape
    normal = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    q = (normal(*shape) * 1.5 + 0.2).to(dtype)
    k = None if kv_heads is None else (normal(*lead, tokens, kv_heads, d) * 0.7).to(dtype)
    dq, dk = normal(*shape).to(dtype), None if k is None else normal(*k.shape).to(dtype)
    wq = (normal(d) * 0.2 + 1).to(dtype) if "q" in weights else None
    wk = (normal(d) * 0.2 + 1).to(dtype) if "k" in weights and k is not None else None
    table = fm.rotary_table(rows or tokens, turned, device=device)
    view = view or (lambda t: t)
    args = dict(q_weight=wq, k_weight=wk, kind=kind, pairing=pairing, eps=EPS)
    vq, vk = view(q), None if k is None else view(k)
    yq, yk = fm.head_rotary_forward(vq, vk, table, positions, **args)
    gq, gk, gwq, gwk = fm.head_rotary_pullback(dq, dk, vq, vk, table, positions, **args)
    at = torch.arange(tokens, device=device) if positions is None else positions.long() - 1
    inside = (at >= 0) & (at < table.shape[0])
    picked = table[torch.where(inside, at, 0)] if table.shape[0] else table.new_zeros(*at.shape, turned)
    picked, inside = picked[..., None, :].expand(*lead, tokens, 1, turned), inside.expand(*lead, tokens)
    for name, x, w, dy, y, gx, gw in (("q", q, wq, dq, yq, gq, gwq), ("k", k, wk, dk, yk, gk, gwk)):
        if x is None:
            assert y is None and gx is None and gw is None
            continue
        want = reference(x, w, picked, turned, kind, pairing, dy, inside)
        close(y, want["y"], name)
        close(gx, want["dx"], "d" + name)
        if w is None:
            assert gw is None
        else:
            close(gw, want["dw"], f"d{name}_weight")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("pairing", ["halves", "neighbours"])
@pytest.mark.parametrize("shape,kv_heads,turned", [
    ((1, 1, 1, 64), 1, 64), ((2, 33, 12, 64), 12, 64), ((3, 7, 9, 50), 3, 36), ((2, 5, 3, 128), 1, 96),
    ((40, 4, 2), 2, 2), ((2, 9, 5, 32), 1, 32), ((6, 3, 512), 2, 512), ((5, 2, 300), 1, 100), ((2, 3, 1, 16), 7, 0),
    ((1, 130, 70, 16), 70, 16), ((3, 4, 96), 2, 64),
])
def test_heads(dtype, kind, pairing, shape, kv_heads, turned, device):
    check(shape, kv_heads, turned, dtype, device, kind, pairing)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weights", ["", "q", "k"])
def test_without_norms(dtype, weights, device):
    """Heads without a weight are only turned."""
    check((2, 20, 4, 64), 2, 64, dtype, device, weights=weights)
    check((2, 20, 4, 34), 2, 20, dtype, device, weights=weights, pairing="neighbours")


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_alone(dtype, device):
    check((2, 20, 4, 64), None, 32, dtype, device)
    check((20, 3, 64), 0, 64, dtype, device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_positions(dtype, id_type, device):
    """Shared or each sequence's own, far ones, and ones that are none of the table's: zeros."""
    g = torch.Generator(device=device).manual_seed(5)
    own = torch.randint(1, 9001, (3, 11), generator=g, device=device).to(id_type)
    check((3, 11, 4, 64), 2, 64, dtype, device, positions=own, rows=9000)
    check((3, 11, 4, 64), 2, 64, dtype, device, positions=own[0].contiguous(), rows=9000)
    own[0, 3], own[1, 0], own[2, 10], own[2, 4] = 0, -5, 9001, 2 ** 31 - 1
    check((3, 11, 4, 64), 2, 64, dtype, device, positions=own, rows=9000)
    check((3, 11, 4, 62), 2, 30, dtype, device, positions=own, rows=9000, kind="layer", pairing="neighbours")
    check((11, 4, 64), 2, 64, dtype, device, positions=own[2].contiguous(), rows=9000)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 48, 30])
def test_strides(dtype, d, device):
    """Heads before tokens, rows apart, and a start that is no 16-byte boundary."""
    check((2, 19, 4, d), 2, d, dtype, device, view=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    check((2, 19, 4, d), 2, d, dtype, device, view=lambda t: torch.cat([t, t + 1], 2)[:, :, :t.shape[2]])
    check((2, 19, 4, d), 2, d, dtype, device,
          view=lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_tokens(dtype, device):
    """More tokens than waves: the weights' sums run over several tokens a wave."""
    check((3, 3001, 4, 64), 4, 64, dtype, device)
    check((9000, 1, 20), 1, 20, dtype, device, kind="layer")


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing(dtype, device):
    check((0, 5, 2, 64), 2, 64, dtype, device)
    check((2, 0, 2, 64), 2, 64, dtype, device, rows=4)
    q = torch.zeros(2, 3, 4, 0, device=device, dtype=dtype)
    y, none = fm.head_rotary_forward(q, None, fm.rotary_table(3, 0, device=device))
    assert y.shape == q.shape and none is None


def test_table():
    t = fm.rotary_table(100_001, 8, base=500.0)
    i = torch.arange(4, dtype=torch.float64)
    angle = 100_000 * 500.0 ** (-2.0 * i / 8)
    # a row's entries are the angles' cosines and sines, rounded (the angle itself is off by 2 units of 2^-53)
    assert (t[-1, :4].double() - angle.cos()).abs().max() <= 2.0 ** -25 + 1e-10
    assert (t[-1, 4:].double() - angle.sin()).abs().max() <= 2.0 ** -25 + 1e-10
    assert t.dtype == torch.float32 and t[0].tolist() == [1.0] * 4 + [0.0] * 4
    for bad in ((-1, 8), (3, 7), (3, -2)):
        with pytest.raises(fm.ArgumentError):
            fm.rotary_table(*bad)


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd_and_differences(dtype, device):
    g = torch.Generator(device=device).manual_seed(8)
    normal = lambda *s: torch.randn(*s, generator=g, device=device).to(dtype)  # noqa: E731
    x = [normal(2, 9, 4, 32), normal(2, 9, 2, 32), normal(32), normal(32)]
    dq, dk = normal(2, 9, 4, 32), normal(2, 9, 2, 32)
    table = fm.rotary_table(9, 32, device=device)
    leaves = [t.clone().requires_grad_() for t in x]
    out = fm.head_rotary(leaves[0], leaves[1], table, q_weight=leaves[2], k_weight=leaves[3])
    torch.autograd.backward(out, (dq, dk))
    args = dict(q_weight=x[2], k_weight=x[3])
    grads = fm.head_rotary_pullback(dq, dk, x[0], x[1], table, **args)
    for leaf, want in zip(leaves, grads):
        assert torch.equal(leaf.grad, want)
    # one output alone: the other's cotangent is zero
    leaves = [t.clone().requires_grad_() for t in x]
    fm.head_rotary(leaves[0], leaves[1], table, q_weight=leaves[2], k_weight=leaves[3])[0].backward(dq)
    assert torch.equal(leaves[0].grad, grads[0]) and torch.equal(leaves[2].grad, grads[2])
    assert not leaves[1].grad.any() and not leaves[3].grad.any()
    if dtype == torch.float32:
        for i, grad in enumerate(grads):
            along = normal(*grad.shape)
            sides = []
            for sign in (1.0, -1.0):
                moved = list(x)
                moved[i] = moved[i] + sign * 0.01 * along
                y = fm.head_rotary_forward(moved[0], moved[1], table, q_weight=moved[2], k_weight=moved[3])
                sides.append(sum((a.double() * b.double()).sum() for a, b in zip(y, (dq, dk))))
            slope = float(sides[0] - sides[1]) / 0.02
            # off by h^2 / 6 of the third derivative, which is of the size of the slope's own terms
            assert abs(slope - float((grad.double() * along.double()).sum())) < 1e-3 * float(grad.norm() * along.norm())


def test_refusals(device):
    q, k = torch.zeros(2, 5, 4, 32, device=device), torch.zeros(2, 5, 2, 32, device=device)
    t = fm.rotary_table(5, 32, device=device)
    one = torch.ones(5, dtype=torch.int32, device=device)
    bad = [
        (fm.ArgumentError, (q.cpu(), k, t), {}), (fm.ArgumentError, (q, k.cpu(), t), {}),
        (fm.ArgumentError, (q, k, t.cpu()), {}), (fm.ArgumentError, (q, k, t.double()), {}),
        (fm.ArgumentError, (q, k.half(), t), {}), (fm.DimensionMismatch, (q, k[:, :4], t), {}),
        (fm.DimensionMismatch, (q, k[..., :16], t), {}), (fm.DimensionMismatch, (q, k, t[:4]), {}),
        (fm.DimensionMismatch, (q, k, fm.rotary_table(5, 34, device=device)), {}),
        (fm.DimensionMismatch, (q[..., :31], k[..., :31], t[:, :30].contiguous()), {}),
        (fm.ArgumentError, (q.transpose(2, 3).contiguous().transpose(2, 3), k, t), {}),
        (fm.ArgumentError, (q, k, t, one.float()), {}), (fm.DimensionMismatch, (q, k, t, one[:4].contiguous()), {}),
        (fm.DimensionMismatch, (q, k, t, one.expand(3, 5).contiguous()), {}),
        (fm.ArgumentError, (q, k, t), dict(kind="batch")), (fm.ArgumentError, (q, k, t), dict(pairing="thirds")),
        (fm.DimensionMismatch, (q, k, t), dict(q_weight=torch.ones(16, device=device))),
        (fm.ArgumentError, (q, k, t), dict(k_weight=torch.ones(32, device=device).half())),
        (fm.UnsupportedError, (q.double(), k.double(), t), {}),
        (fm.UnsupportedError, (torch.zeros(5, 1, 514, device=device), None, t), {}),
    ]
    for error, arrays, options in bad:
        with pytest.raises(error):
            fm.head_rotary_forward(*arrays, **options)
