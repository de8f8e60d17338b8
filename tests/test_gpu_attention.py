"""Attention over heads and its pullback against their definition in 64 bits (attention_reference.py),
with bounds for every entry."""
import pytest
import torch

import flashmaxsim as fm
from attention_reference import check, counts, reference

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(shape_q, shape_k, dtype, device, seed=0, size=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    q, k, v = normal(*shape_q) * size, normal(*shape_k), normal(*shape_k)
    return [t.to(dtype) for t in (q, k, v, normal(*shape_q))]


def padded(q, k, v, do, qmask=None, kmask=None, causal=False, window=None, scale=None, view=None):
    """Both calls on a padded batch, every sequence checked."""
    scale_ = q.shape[-1] ** -0.5 if scale is None else scale
    args = dict(causal=causal, window=window, scale=scale)
    view = view or (lambda t: t)
    o, kept = fm.attention_forward(view(q), view(k), view(v), qmask, kmask, keep=True, **args)
    plain = fm.attention_forward(view(q), view(k), view(v), qmask, kmask, **args)
    assert torch.equal(o, plain)  # (what is kept changes nothing)
    grads = fm.attention_pullback(do, view(q), view(k), view(v), o, kept, qmask, kmask, **args)
    for b in range(q.shape[0]):
        keep = counts(q.shape[1], k.shape[1], causal, window, q.device)
        if qmask is not None:
            keep = keep & qmask[b][:, None]
        if kmask is not None:
            keep = keep & kmask[b][None]
        want = reference(q[b], k[b], v[b], keep, scale_, do[b])
        for name, x in zip(("o", "dq", "dk", "dv"), (o, *grads)):
            check(x[b], want[name], f"{name} of sequence {b}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,d", [
    (1, 1, 1, 1, 1, 32), (2, 1, 77, 2, 2, 64), (1, 32, 32, 3, 3, 64), (2, 33, 65, 2, 1, 32),
    (1, 129, 64, 2, 2, 128), (2, 63, 191, 6, 2, 96), (1, 200, 130, 4, 4, 80), (3, 5, 3, 12, 4, 16),
    (1, 70, 70, 2, 2, 17), (2, 40, 41, 3, 1, 50), (1, 257, 300, 1, 1, 128), (1, 3, 200, 5, 1, 1),
])
def test_padded(dtype, B, Tq, Tk, H, Hk, d, device):
    padded(*inputs((B, Tq, H, d), (B, Tk, Hk, d), dtype, device, seed=Tq * 1000 + d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal,window", [(True, None), (False, 0), (False, 20), (True, 33), (True, 0),
                                           (False, 10 ** 9)])
@pytest.mark.parametrize("Tq,Tk,H,Hk", [(130, 130, 2, 2), (150, 70, 4, 2), (65, 200, 3, 1)])
def test_positions(dtype, causal, window, Tq, Tk, H, Hk, device):
    """With more queries than keys the first queries see nothing."""
    padded(*inputs((1, Tq, H, 64), (1, Tk, Hk, 64), dtype, device, seed=Tq), causal=causal, window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 30)])
def test_masks(dtype, causal, window, device):
    """Padding of both sides, scattered masks, a sequence without keys, and one without queries; what is
    masked holds NaN and infinities."""
    B, Tq, Tk, H, Hk, d = 5, 150, 170, 4, 2, 64
    q, k, v, do = inputs((B, Tq, H, d), (B, Tk, Hk, d), dtype, device, seed=3)
    g = torch.Generator(device=device).manual_seed(4)
    qmask = torch.rand(B, Tq, generator=g, device=device) < 0.6
    kmask = torch.rand(B, Tk, generator=g, device=device) < 0.5
    qmask[0], kmask[0] = torch.arange(Tq, device=device) < 97, torch.arange(Tk, device=device) < 65
    kmask[1] = False
    qmask[2] = False
    kmask[3, :64], kmask[3, 128:] = False, False
    for t, m in ((q, qmask), (k, kmask), (v, kmask), (do, qmask)):
        t[~m] = float("nan")
    v[~kmask & (torch.rand(B, Tk, generator=g, device=device) < 0.5)] = float("inf")
    padded(q, k, v, do, qmask, kmask, causal, window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_mask(dtype, device):
    q, k, v, do = inputs((2, 40, 2, 32), (2, 90, 2, 32), dtype, device)
    mask = torch.arange(90, device=device)[None] < torch.tensor([[50], [90]], device=device)
    padded(q, k, v, do, kmask=mask)
    padded(q, k, v, do, qmask=mask[:, :40].contiguous())
    bytes_ = mask.to(torch.uint8) * 7
    assert torch.equal(fm.attention_forward(q, k, v, kmask=bytes_), fm.attention_forward(q, k, v, kmask=mask))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_long_mask(dtype, device):
    """More keys, and more query rows, than mask bits are held at a time."""
    n = 16384 + 150
    g = torch.Generator(device=device).manual_seed(1)
    mask = torch.rand(1, n, generator=g, device=device) < 0.3
    mask[:, 5000:12000] = False
    padded(*inputs((1, 3, 2, 32), (1, n, 1, 32), dtype, device), kmask=mask)
    padded(*inputs((1, n, 2, 32), (1, 5, 1, 32), dtype, device), qmask=mask)
    padded(*inputs((1, n, 1, 32), (1, 70, 1, 32), dtype, device), causal=True, qmask=mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,d,causal,window", [
    (1, 1, 5000, 4, 1, 128, False, None), (2, 1, 3001, 2, 2, 64, True, None), (1, 40, 2500, 6, 2, 32, True, 300),
    (1, 130, 1100, 1, 1, 96, False, 5), (1, 1, 257, 1, 1, 64, False, None), (1, 2, 4096, 1, 1, 20, False, 0),
])
def test_split(dtype, B, Tq, Tk, H, Hk, d, causal, window, device):
    """Few rows and many keys: the keys are split among workgroups, some of which have none that count."""
    q, k, v, do = inputs((B, Tq, H, d), (B, Tk, Hk, d), dtype, device, seed=Tk)
    padded(q, k, v, do, causal=causal, window=window)
    mask = torch.zeros(B, Tk, dtype=torch.bool, device=device)
    mask[0, 100:180] = True
    k[~mask] = float("nan")
    padded(q, k, v, do, kmask=mask, causal=causal, window=window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_split_ragged(dtype, device):
    ragged([1, 0, 3], [3000, 700, 0], 4, 2, 64, dtype, device)
    ragged([2, 2], [1200, 5], 2, 2, 64, dtype, device, causal=True, front=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_scale(dtype, scale, device):
    padded(*inputs((1, 70, 2, 64), (1, 100, 1, 64), dtype, device, size=0.5), scale=scale, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_key_has_the_weight(dtype, device):
    """Scores spread over tens: p nearly one and the rest small, dp - delta a difference of near equals."""
    padded(*inputs((1, 100, 2, 64), (1, 120, 2, 64), dtype, device, size=6.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e-6, 1e-3, 300.0])
def test_cotangents_of_any_size(dtype, size, device):
    """A large part of fp16's range, token by token as well."""
    q, k, v, do = inputs((1, 130, 2, 64), (1, 140, 2, 64), dtype, device)
    padded(q, k, v, (do.float() * size).to(dtype))
    spread = 10.0 ** (torch.arange(130, device=device) % 5 - 2).float()
    padded(q, k, v, (do.float() * spread[None, :, None, None]).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 40, 30])
def test_strides(dtype, d, device):
    """Slices of one projection's output, heads before tokens, rows apart, and a broadcast batch."""
    g = torch.Generator(device=device).manual_seed(2)
    B, T, H, Hk = 2, 75, 4, 2
    qkv = torch.randn(B, T, H + 2 * Hk, d, generator=g, device=device).to(dtype)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    do = torch.randn(B, T, H, d, generator=g, device=device).to(dtype)
    padded(q, k, v, do, causal=True)
    swap = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    padded(q, k, v, do, view=swap)
    apart = lambda t: torch.stack([t, t + 1], 2)[:, :, 0]  # noqa: E731
    padded(q, k, v, do, view=apart)
    one = k[:1].expand(B, -1, -1, -1)
    padded(q, one, v, do)
    # 2-byte steps from a 16-byte boundary
    off = torch.empty(k.numel() + 1, dtype=dtype, device=device)[1:].view(k.shape).copy_(k)
    padded(q, off, v, do)


def ragged(lens_q, lens_k, H, Hk, d, dtype, device, causal=False, window=None, front=0, behind=0, most=None):
    """front, behind: token rows before the first sequence and after the last."""
    cus = [torch.tensor([1 + front + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)
           for lens in (lens_q, lens_k)]
    nq, nk = (front + sum(n) + behind for n in (lens_q, lens_k))
    q, k, v, do = inputs((nq, H, d), (nk, Hk, d), dtype, device, seed=9)
    inside = []
    for n, lens in ((nq, lens_q), (nk, lens_k)):
        at = torch.arange(n, device=device)
        inside.append((at >= front) & (at < front + sum(lens)))
    for t, m in ((q, inside[0]), (do, inside[0]), (k, inside[1]), (v, inside[1])):
        t[~m] = float("nan")
    mq, mk = most or (max(lens_q, default=0), max(lens_k, default=0))
    args = dict(cu_q=cus[0], cu_k=cus[1], max_q=mq, max_k=mk, causal=causal, window=window)
    o, kept = fm.attention_forward(q, k, v, keep=True, **args)
    grads = fm.attention_pullback(do, q, k, v, o, kept, **args)
    at_q = at_k = front
    for a, b in zip(lens_q, lens_k):
        s, t = slice(at_q, at_q + a), slice(at_k, at_k + b)
        want = reference(q[s], k[t], v[t], counts(a, b, causal, window, device), d ** -0.5, do[s])
        for name, x, part in zip(("o", "dq", "dk", "dv"), (o, *grads), (s, s, t, t)):
            check(x[part], want[name], f"{name} of tokens {part}")
        at_q, at_k = at_q + a, at_k + b
    for x, m in zip((o, *grads), (inside[0], inside[0], inside[1], inside[1])):
        assert not x[~m].any()  # rows of no sequence: zeros


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 16)])
def test_ragged(dtype, causal, window, device):
    lens = [5, 0, 130, 1, 64, 65, 33]
    ragged(lens, lens, 4, 2, 64, dtype, device, causal, window)
    ragged(lens, [70, 3, 0, 1, 200, 64, 31], 3, 3, 32, dtype, device, causal, window, front=3, behind=70)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ragged_odd(dtype, device):
    ragged([31, 100], [31, 100], 3, 1, 20, dtype, device, True, front=1, behind=2)
    ragged([31, 100], [31, 100], 2, 2, 64, dtype, device, most=(131, 131))  # lengths not known
    ragged([], [], 2, 2, 64, dtype, device, behind=5)
    ragged([0, 0], [0, 0], 2, 2, 64, dtype, device, behind=5)


def test_bad_cu(device):
    """A cu that decreases or leaves the tokens is clamped: other sequences keep their results."""
    q, k, v, _ = inputs((100, 2, 64), (100, 2, 64), torch.bfloat16, device)
    good = torch.tensor([1, 31, 61, 101], dtype=torch.int32, device=device)
    want = fm.attention_forward(q, k, v, cu_q=good, cu_k=good, max_q=40, max_k=40)
    for bad in ([1, 31, 61, 5000], [1, 31, 61, 2 ** 31 - 1], [1, 31, 61, 40], [1, 31, 61, -7]):
        cu = torch.tensor(bad, dtype=torch.int32, device=device)
        got = fm.attention_forward(q, k, v, cu_q=cu, cu_k=cu, max_q=40, max_k=40)
        assert torch.equal(got[:60], want[:60])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nothing(dtype, device):
    """No keys, no queries, no sequences, no heads, no values."""
    for sq, sk in (((2, 7, 2, 64), (2, 0, 2, 64)), ((2, 0, 2, 64), (2, 7, 2, 64)), ((0, 7, 2, 64), (0, 7, 2, 64)),
                   ((2, 7, 0, 64), (2, 7, 0, 64)), ((2, 7, 2, 0), (2, 7, 2, 0))):
        q, k, v, do = inputs(sq, sk, dtype, device)
        o, kept = fm.attention_forward(q, k, v, keep=True)
        grads = fm.attention_pullback(do, q, k, v, o, kept)
        for x, like in zip((o, *grads), (q, q, k, v)):
            assert x.shape == like.shape and not x.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_not_finite(dtype, device):
    """A NaN reaches the rows that it belongs to, and no other sequence or head."""
    q, k, v, do = inputs((2, 40, 2, 64), (2, 90, 2, 64), dtype, device)
    q[0, 3, 1, 5] = float("nan")
    k[1, 70, 0, 2] = float("nan")
    o = fm.attention_forward(q, k, v)
    bad = torch.isnan(o)
    assert bad[0, 3, 1].all() and int(bad[0].sum()) == 64
    assert bad[1, :, 0].all() and not bad[1, :, 1].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd_and_differences(dtype, device):
    """Autograd's gradients are the pullback's, and the pullback's are those of differences."""
    q, k, v, do = inputs((2, 20, 4, 32), (2, 30, 2, 32), dtype, device)
    mask = torch.arange(30, device=device)[None] < torch.tensor([[17], [30]], device=device)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = fm.attention(*leaves, None, mask, window=12)
    o.backward(do)
    o2, kept = fm.attention_forward(q, k, v, None, mask, window=12, keep=True)
    grads = fm.attention_pullback(do, q, k, v, o2, kept, None, mask, window=12)
    assert torch.equal(o, o2)
    for leaf, g in zip(leaves, grads):
        assert torch.equal(leaf.grad, g)
    if dtype == torch.float32:
        # central differences along a random direction of each input: off by h^2 and by o's own rounding / h
        for i, g in enumerate(grads):
            d = torch.randn(g.shape, generator=torch.Generator(device=device).manual_seed(i), device=device)
            sides = []
            for sign in (1.0, -1.0):
                moved = [q, k, v]
                moved[i] = moved[i] + sign * 0.01 * d
                sides.append((fm.attention_forward(*moved, None, mask, window=12).double() * do.double()).sum())
            slope = float((sides[0] - sides[1]) / 0.02)
            assert abs(slope - float((g.double() * d.double()).sum())) < 2e-3 * float(g.double().norm() * d.double().norm()) / 8
    with torch.no_grad():
        assert torch.equal(fm.attention(*leaves, None, mask, window=12), o)


def test_second_derivatives_are_refused(device):
    q = torch.randn(1, 8, 1, 32, device=device, requires_grad=True)
    g, = torch.autograd.grad(fm.attention(q, q, q).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals(device):
    q, k, v, _ = inputs((2, 8, 4, 32), (2, 8, 2, 32), torch.bfloat16, device)
    cu = torch.tensor([1, 9], dtype=torch.int32, device=device)
    bad = [
        (fm.ArgumentError, (q.cpu(), k, v), {}),
        (fm.ArgumentError, (q, k.cpu(), v), {}),
        (fm.ArgumentError, (q, k.half(), v.half()), {}),
        (fm.DimensionMismatch, (q, k, v[:, :4]), {}),
        (fm.DimensionMismatch, (q, k[:1], v[:1]), {}),
        (fm.DimensionMismatch, (q[..., :16], k, v), {}),
        (fm.DimensionMismatch, (q[:, :, :3], k, v), {}),
        (fm.ArgumentError, (q.transpose(2, 3).contiguous().transpose(2, 3), k, v), {}),
        (fm.DimensionMismatch, (q, k, v), dict(kmask=torch.ones(2, 9, dtype=torch.bool, device=device))),
        (fm.ArgumentError, (q, k, v), dict(kmask=torch.ones(2, 8, device=device))),
        (fm.ArgumentError, (q, k, v), dict(kmask=torch.ones(2, 8, dtype=torch.bool))),
        (fm.ArgumentError, (q, k, v), dict(window=-1)),
        (fm.ArgumentError, (q, k, v), dict(max_q=8)),
        (fm.DimensionMismatch, (q, k, v), dict(cu_q=cu, cu_k=cu)),
        (fm.ArgumentError, (q[0], k[0], v[0]), dict(cu_q=cu)),
        (fm.ArgumentError, (q[0], k[0], v[0]), dict(cu_q=cu.long(), cu_k=cu)),
        (fm.DimensionMismatch, (q[0], k[0], v[0]), dict(cu_q=cu, cu_k=cu[:1])),
        (fm.ArgumentError, (q[0], k[0], v[0]), dict(cu_q=cu, cu_k=cu, kmask=torch.ones(8, dtype=torch.bool, device=device))),
        (fm.UnsupportedError, tuple(torch.zeros(1, 4, 1, 136, device=device) for _ in range(3)), {}),
        (fm.UnsupportedError, tuple(torch.zeros(1, 4, 1, 32, device=device, dtype=torch.float64) for _ in range(3)), {}),
    ]
    for error, arrays, options in bad:
        with pytest.raises(error):
            fm.attention_forward(*arrays, **options)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Tq,Tk", [(0, 5), (5, 0), (0, 0)])
def test_no_tokens(dtype, Tq, Tk, device):
    """Without queries the keys' gradients are zero, without keys the results are."""
    q, k, v, do = inputs((2, Tq, 4, 48), (2, Tk, 2, 48), dtype, device)
    o, kept = fm.attention_forward(q, k, v, keep=True)
    for t, like in zip((o, *fm.attention_pullback(do, q, k, v, o, kept)), (q, q, k, v)):
        assert t.shape == like.shape and not t.any()


def test_sizes_past_64_bits(device):
    q, k, v, do = inputs((70, 2, 32), (70, 2, 32), torch.bfloat16, device)
    cu = torch.tensor([1, 31, 71], dtype=torch.int32, device=device)
    whole = fm.attention_forward(q, k, v, cu_q=cu, cu_k=cu)
    for args in (dict(window=10 ** 30), dict(window=2 ** 64)):
        assert torch.equal(fm.attention_forward(q, k, v, cu_q=cu, cu_k=cu, **args), whole)
    with pytest.raises(fm.UnsupportedError):
        fm.attention_forward(q, k, v, cu_q=cu, cu_k=cu, max_q=2 ** 64 + 70, max_k=70)
