"""How far a value that is not finite reaches in attention's results and gradients: not into other sequences or key heads,
and under a window not past the tiles of 64 keys and 64 query rows that it lies in."""
import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
B, T, H, HK, D, WINDOW, AT = 2, 700, 4, 2, 64, 20, 350


def run(x, **args):
    q, k, v, do = x
    o, kept = fm.attention_forward(q, k, v, keep=True, **args)
    return (o, *fm.attention_pullback(do, q, k, v, o, kept, **args))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("causal", [False, True])
def test_reach(dtype, which, value, causal, device):
    g = torch.Generator(device=device).manual_seed(7)
    x = [(torch.randn(B, T, n, D, generator=g, device=device) * s).to(dtype) for n, s in ((H, 1), (HK, 1), (HK, 3), (H, 3))]
    good = run(x, window=WINDOW, causal=causal)
    i = "q k v do".split().index(which)
    head = 0  # (query heads 0 and 1 share key head 0)
    x[i] = x[i].clone()
    x[i][0, AT, head, 5] = value
    got = run(x, window=WINDOW, causal=causal)
    # a query's tile of keys, or a key's of query rows, ends at most 63 from what it reaches; a key's gradient takes in
    # queries that saw a bad key: twice the window, and 32 rows of a wave on each side
    far = 2 * (WINDOW + 64 + 32)
    for name, a, b in zip(("o", "dq", "dk", "dv"), got, good):
        n = a.shape[2] // HK  # query heads of a key head
        clean = torch.ones(a.shape[:3], dtype=torch.bool, device=device)
        clean[0, AT - far:AT + far, :n] = False
        assert torch.isfinite(a[clean]).all(), name
        # (fp16: the scale that ds takes is of the finite rows)
        torch.testing.assert_close(a[clean], b[clean])
        assert clean[0, :, :n].any()
    assert not all(torch.isfinite(a).all() for a in got)
