"""Attention of scores from ten to ten thousand million, which are whole multiples of a power of two: every sum of products
is exact in 32 bits, whatever its order, so that only the softmax and what follows it can be off.

A weight exp2(t) / l, t = (x - max) scale log2 e, may be off by t's own roundings (the factor's and the product's,
|t| 2^-23), the exponential's (2^-23) and those of a sum of as many terms as there are keys; nothing in that grows
with the scores themselves."""
import math

import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = 2.0 ** -24
# base-2 logarithms of q's and k's common factors, how many bits below the score its steps lie, the scale
SCORES = {"10": (2, 4, 2.0 ** -5), "1e3": (4, 11, 2.0 ** -3), "3e4": (4, 16, 2.0 ** 2), "4e6": (4, 22, 2.0 ** 8),
          "1e8": (12, 20, 2.0 ** -2), "3e10": (15, 23, 1.0)}
SMALL = {"2^-108": (60, 20, 2.0 ** -108)}  # a small scale of scores near the end of the range (not in fp16)
SHAPES = [(70, 100, 2, 2, 64), (130, 90, 4, 2, 128), (1, 3000, 2, 1, 64), (33, 70, 2, 2, 40)]


def inputs(name, Tq, Tk, H, Hk, d, dtype, device):
    factor, bits, scale = (SCORES | SMALL)[name]
    top = 5 + 2 * factor  # 32 products of 2^factor 2^factor
    g = torch.Generator(device=device).manual_seed(bits)
    q, k = torch.zeros(1, Tq, H, d, device=device), torch.zeros(1, Tk, Hk, d, device=device)
    q[..., :32], k[..., :32] = 2.0 ** factor, 2.0 ** factor
    whole = lambda n, *s: torch.randint(0, n, s, generator=g, device=device)  # noqa: E731
    q[..., 32] = 2.0 ** (top - bits) * (1 + whole(2, 1, Tq, H))
    k[..., 32] = whole(8, 1, Tk, Hk).float()
    normal = lambda t: torch.randn(t.shape, generator=g, device=device)  # noqa: E731
    made = [t.to(dtype) for t in (q, k, normal(k), normal(q) * 0.02)]
    assert torch.equal(made[0].float(), q) and torch.equal(made[1].float(), k)
    return *made, scale


def weights(q, k, scale, dtype):
    """Weights (heads, Tq, Tk) in 64 bits, and how far off they may be, relative to themselves."""
    s = (q @ k.transpose(1, 2).contiguous()) * scale
    assert torch.equal((s / scale).float().double(), s / scale)
    t = (s - s.amax(-1, keepdim=True)) * math.log2(math.e)
    p = torch.exp2(t)
    p = p / p.sum(-1, keepdim=True)
    own = math.log(2) * t.abs() * 2.0 ** -23 + 2.0 ** -22
    # (16 bits, pullback: the sum goes in as its logarithm, of 12 at most, rounded twice)
    own = own + (0 if dtype == torch.float32 else 2 * math.log(2) * 12 * UNIT)
    return p, own + (p * own).sum(-1, keepdim=True) + UNIT * (k.shape[1] + 8)


def wide(t, group=1):
    return t[0].double().transpose(0, 1).repeat_interleave(group, 0)


def close(got, want, far, what):
    half = torch.finfo(got.dtype).eps / 2
    far = half * want.abs() + 1.01 * far + torch.finfo(got.dtype).smallest_normal * half
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} entries are not finite"
    over = float(((wide(got) - want).abs() / far).max())
    assert over <= 1.0, f"{what}: {over:.3f} times as far off as roundings may be"


def rounding(dtype):
    """Of a weight on its way into a product (16 bits: two values), relative; and its grid in fp16."""
    half = torch.finfo(dtype).eps / 2
    return (half * half * 1.01 if dtype != torch.float32 else 0.0), (2.0 ** -35 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", SCORES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(dtype, name, shape, device):
    q, k, v, _, scale = inputs(name, *shape, dtype, device)
    group = shape[2] // shape[3]
    p, off = weights(wide(q), wide(k, group), scale, dtype)
    V = wide(v, group)
    rough, grid = rounding(dtype)
    o = fm.attention_forward(q, k, v, scale=scale)
    close(o, p @ V, ((off + rough) * p) @ V.abs() + grid * V.abs().sum(1, keepdim=True), "o")
    assert torch.equal(o, fm.attention_forward(-q, k, v, scale=-scale))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", SCORES)
@pytest.mark.parametrize("shape", SHAPES)
def test_pullback(dtype, name, shape, device):
    """ds = p (dp - delta): dp and delta are sums over a head's values, delta of the output, which in 16 bits
    comes with what its rounding left."""
    q, k, v, do, scale = inputs(name, *shape, dtype, device)
    Tq, Tk, H, Hk, d = shape
    group = H // Hk
    p, off = weights(wide(q), wide(k, group), scale, dtype)
    Q, K, V, D = wide(q), wide(k, group), wide(v, group), wide(do)
    rough, grid = rounding(dtype)
    half = torch.finfo(dtype).eps / 2
    dp = D @ V.transpose(1, 2).contiguous()
    dp_size = D.abs() @ V.abs().transpose(1, 2).contiguous()
    delta, delta_size = (p * dp).sum(-1, keepdim=True), (p * dp_size).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    left = half if dtype == torch.float32 else 4 * half * half
    delta_off = (UNIT * (d + 8) + left + rough) * delta_size + (off * p * dp_size).sum(-1, keepdim=True) \
        + grid * dp_size.sum(-1, keepdim=True)
    ds_off = p * (UNIT * (d + 8) * dp_size + delta_off) + (off + rough) * ds.abs()
    if dtype == torch.float16:  # ds on its grid: 2^15 p times a factor that brings 2 |do| |v| to 1/2 at least
        ds_off = ds_off + 4 * D.norm(dim=-1).amax() * V.norm(dim=-1).amax() * 2.0 ** -40
    sums = UNIT * (Tq * group + Tk)
    turned = lambda t: t.transpose(1, 2).contiguous()  # noqa: E731
    share = lambda t: t.view(Hk, group, *t.shape[1:]).sum(1)  # noqa: E731
    o, kept = fm.attention_forward(q, k, v, scale=scale, keep=True)
    dq, dk, dv = fm.attention_pullback(do, q, k, v, o, kept, scale=scale)
    close(dq, scale * ds @ K, scale * ((ds_off + sums * ds.abs()) @ K.abs()), "dq")
    close(dk, share(scale * turned(ds) @ Q), share(scale * turned(ds_off + sums * ds.abs()) @ Q.abs()), "dk")
    close(dv, share(turned(p) @ D), share(turned((off + rough + sums) * p + grid) @ D.abs()), "dv")
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), (lambda x: (-x[0], x[1], x[2]))(
        fm.attention_pullback(do, -q, k, v, o, kept, scale=-scale))))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_small_scale(dtype, shape, device):
    test_forward(dtype, "2^-108", shape, device)
    test_pullback(dtype, "2^-108", shape, device)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_number_for_a_scale(dtype, device):
    q, k, v, do, _ = inputs("10", 33, 70, 2, 2, 40, dtype, device)
    o, kept = fm.attention_forward(q, k, v, scale=float("nan"), keep=True)
    assert all(torch.isnan(t).all() for t in (o, *fm.attention_pullback(do, q, k, v, o, kept, scale=float("nan"))))
    mask = torch.zeros(1, 70, dtype=torch.bool, device=device)
    assert not fm.attention_forward(q, k, v, kmask=mask, scale=float("nan")).any()
