"""The token lookup and its gradient against their definition in 64 bits.

The lookup is one product in fp32 and one rounding; a gradient's entry is a sum of as many terms in fp32 as
its id has tokens, one product and one rounding.  Every entry is held to what those may cost."""
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = 2.0 ** -24


def floor(dtype):
    """Half a step among the type's smallest numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check(ids, vocabulary, dim, dtype, device, scale=1.0, seed=0, shift=0):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        flat = torch.randn(shape[0] * shape[1] + shift, generator=g, device=device).to(dtype)
        return flat[shift:].view(shape)  # (shift: not from a 16-byte boundary)

    weight, de = normal(vocabulary, dim), normal(ids.numel(), dim)
    e = fm.embed_tokens_forward(ids, weight, scale)
    dw = fm.embed_tokens_pullback(de.view(*ids.shape, dim), ids, vocabulary, scale)
    assert e.shape == (*ids.shape, dim) and e.dtype == dtype
    assert dw.shape == (vocabulary, dim) and dw.dtype == dtype
    half = torch.finfo(dtype).eps / 2
    flat = ids.flatten().long()
    real = (flat >= 1) & (flat <= vocabulary)
    at = torch.where(real, flat - 1, 0)
    scale = torch.tensor(scale, dtype=torch.float32).item()
    if vocabulary:
        want = torch.where(real[:, None], weight.double()[at] * scale, 0.0).view(e.shape)
        assert ((e.double() - want).abs() <= (half + UNIT) * 1.001 * want.abs() + floor(dtype)).all()
        assert not e.view(ids.numel(), dim)[~real].any()
    else:
        assert not e.any()
    rows = torch.zeros(vocabulary, dim, dtype=torch.float64, device=device)
    size, count = rows.clone(), torch.zeros(vocabulary, device=device, dtype=torch.float64)
    rows.index_add_(0, at[real], de.double()[real])
    size.index_add_(0, at[real], de.double().abs()[real])
    count.index_add_(0, at[real], torch.ones_like(at[real], dtype=torch.float64))
    want = rows * scale
    bound = half * 1.001 * want.abs() + (count[:, None] + 2) * UNIT * size * abs(scale) + floor(dtype)
    assert ((dw.double() - want).abs() <= bound).all()
    assert not dw[count == 0].any()
    assert torch.equal(dw, fm.embed_tokens_pullback(de.view(*ids.shape, dim), ids, vocabulary, scale))


def zipf(shape, vocabulary, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    u = torch.rand(shape, generator=g, device=device, dtype=torch.float64)
    return (vocabulary ** u).long().clamp(1, vocabulary)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,vocabulary,dim", [
    (1, 1, 8), (3, 7, 64), (32, 500, 768), (1000, 300, 128), (2000, 5000, 1032), (700, 40, 531), (129, 130, 1),
    (65, 1, 24), (4100, 3, 136), (64, 1, 2500),
])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_tokens(dtype, tokens, vocabulary, dim, id_type, device):
    """Few tokens to an id and many (the runs that one wave adds up end at 64), odd widths."""
    check(zipf((tokens,), vocabulary, device).to(id_type), vocabulary, dim, dtype, device, scale=3.7)


@pytest.mark.parametrize("dtype", TYPES)
def test_padding_and_bad_ids(dtype, device):
    ids = zipf((4, 90), 50, device, seed=1)
    ids[:, 70:] = 0
    ids[0, 3], ids[1, 5], ids[2, 7] = -4, 51, 2 ** 40
    check(ids, 50, 96, dtype, device, scale=-0.5)
    check(torch.zeros(3, 5, dtype=torch.int32, device=device), 20, 64, dtype, device)


@pytest.mark.parametrize("runs", [(63, 64, 65), (64,), (65, 1, 0, 200), (3000,)])
def test_runs(runs, device):
    """Runs about the length that one wave takes, scattered over the tokens."""
    ids = torch.cat([torch.full((n,), i + 1) for i, n in enumerate(runs)])
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(2))].to(device)
    check(ids, len(runs), 200, torch.float32, device)
    check(ids, len(runs) + 300, 200, torch.bfloat16, device)


def test_more_tokens_than_bits(device):
    """More tokens than a workgroup's map has bits for."""
    n = (1 << 18) + 5000
    ids = zipf((n,), 200, device, seed=3)
    ids[::2] = 17
    check(ids, 200, 16, torch.float32, device)


@pytest.mark.parametrize("dtype", TYPES)
def test_alignment(dtype, device):
    check(zipf((300,), 70, device), 70, 64, dtype, device, shift=1)


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing(dtype, device):
    none = torch.zeros(0, dtype=torch.int32, device=device)
    check(none, 10, 64, dtype, device)
    check(none, 0, 64, dtype, device)
    check(torch.ones(5, dtype=torch.int32, device=device), 0, 64, dtype, device)
    check(torch.ones(5, dtype=torch.int32, device=device), 9, 0, dtype, device)


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(dtype, device):
    weight = torch.randn(60, 48, device=device).to(dtype).requires_grad_()
    ids = zipf((3, 40), 60, device)
    e = fm.embed_tokens(ids, weight, 2.0)
    de = torch.randn_like(e)
    e.backward(de)
    assert torch.equal(weight.grad, fm.embed_tokens_pullback(de, ids, 60, 2.0))
    # linear in the table: the slope along any direction is the inner product with the gradient
    along = torch.randn_like(weight)
    slope = (fm.embed_tokens_forward(ids, along, 2.0).double() * de.double()).sum()
    got = (weight.grad.double() * along.double()).sum()
    # half a step for each e and each gradient entry, sums of up to 120 terms
    half = torch.finfo(dtype).eps / 2 + 130 * UNIT
    size = (fm.embed_tokens_forward(ids, along.abs(), 2.0).double() * de.double().abs()).sum()
    assert abs(float(slope - got)) <= 2.1 * half * float(size)
    leaf = weight.detach().clone().requires_grad_()
    g, = torch.autograd.grad(fm.embed_tokens(ids, leaf).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals(device):
    weight = torch.zeros(5, 8, device=device)
    ids = torch.ones(3, dtype=torch.int32, device=device)
    for error, args in [
        (fm.ArgumentError, (ids.cpu(), weight)), (fm.ArgumentError, (ids, weight.cpu())),
        (fm.ArgumentError, (ids.float(), weight)), (fm.ArgumentError, (ids, weight.t())),
        (fm.ArgumentError, (ids.to(torch.int16), weight)), (fm.DimensionMismatch, (ids, weight[0])),
        (fm.UnsupportedError, (ids, weight.double())),
        (fm.ArgumentError, (torch.ones(6, dtype=torch.int32, device=device)[::2], weight)),
    ]:
        with pytest.raises(error):
            fm.embed_tokens_forward(*args)
    for error, args in [
        (fm.DimensionMismatch, (torch.zeros(4, 8, device=device), ids, 5)),
        (fm.DimensionMismatch, (torch.zeros(8, device=device), ids, 5)),
        (fm.DimensionMismatch, (torch.zeros(3, 8, device=device), ids, -1)),
        (fm.ArgumentError, (torch.zeros(3, 8), ids, 5)),
        (fm.UnsupportedError, (torch.zeros(3, 8, device=device).double(), ids, 5)),
    ]:
        with pytest.raises(error):
            fm.embed_tokens_pullback(*args)
