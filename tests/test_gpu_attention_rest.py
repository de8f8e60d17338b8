"""What the forward keeps of its output's rounding: the output and what it left are together as exact as the fp32
sums behind them, also where those lie next to the middle between two 16-bit values."""
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,by", [(torch.float16, 2048.0), (torch.bfloat16, 1.0)])
@pytest.mark.parametrize("B,Tq,Tk,d", [(8, 1000, 20, 64), (8, 1000, 20, 128), (8, 1000, 20, 40), (1, 100, 2000, 128)])
def test_what_the_rounding_left(dtype, by, B, Tq, Tk, d, device):
    """(The last shape's keys are split among workgroups.)  Queries of zero: every weight is 1 / Tk and exact but for one
    rounding, the sum of values is off by Tk units at most, the quotient by one; the rest is rounded itself."""
    g = torch.Generator(device=device).manual_seed(d)
    k, v = (torch.randn(B, Tk, 2, d, generator=g, device=device).to(dtype) for _ in range(2))
    q = torch.zeros(B, Tq, 2, d, device=device, dtype=dtype)
    # (another mean for each query: the first keys that it sees)
    o, kept = fm.attention_forward(q, k, v, causal=True, keep=True)
    seen = (torch.arange(Tq, device=device) + Tk - Tq + 1).clamp(min=0)
    sums = torch.cat([torch.zeros(B, 1, 2, d, device=device, dtype=torch.float64), v.double().cumsum(1)], 1)
    size = torch.cat([torch.zeros(B, 1, 2, d, device=device, dtype=torch.float64), v.double().abs().cumsum(1)], 1)
    n = seen.clamp(min=1).double()[:, None, None]
    want, size = sums[:, seen] / n, size[:, seen] / n
    half = torch.finfo(dtype).eps / 2
    got = o.double() + kept.rest.double() / by
    far = (Tk + 4) * 2.0 ** -24 * size + 1.01 * half * half * want.abs() + torch.finfo(dtype).smallest_normal * half / by
    assert ((got - want).abs() <= far).all(), float(((got - want).abs() / far).nan_to_num(0).max())
    assert ((o.double() - want).abs() <= 1.01 * half * want.abs() + far + torch.finfo(dtype).smallest_normal * half).all()
