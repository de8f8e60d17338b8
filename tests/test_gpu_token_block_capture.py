"""The token block's calls under graph capture without lent workspace: they fail, add nothing to the
graph and leave the capture as it was; outside capture they take the library's pool."""
import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import _lib, boundary

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_lender(device):
    boundary._this_thread()
    _lib.lib().fms_set_workspace_lender(_lib.LENDER(0))
    yield
    boundary._this_thread()  # the drivers' lender again


@pytest.mark.parametrize("declines", [False, True])
def test_captured_calls_are_lent_workspace_or_fail(device, no_lender, declines):
    lender = _lib.LENDER(lambda nbytes, stream: None)
    if declines:
        _lib.lib().fms_set_workspace_lender(lender)
    g = torch.Generator(device=device).manual_seed(0)
    x, dh = (torch.randn(40, n, generator=g, device=device) for n in (51, 64))  # rows of 204 bytes: copied
    wg, wu = (torch.randn(64, 51, generator=g, device=device) for _ in range(2))
    w = torch.ones(51, device=device)
    calls = (lambda: fm.gated_ffn_forward(x, wg, wu), lambda: fm.gated_ffn_pullback(dh, x, wg, wu),
             lambda: fm.block_norm_pullback(None, x, x, pre_weight=w))
    eager = [call() for call in calls]  # from the pool
    graph, y = torch.cuda.CUDAGraph(), torch.zeros(8, device=device)
    with torch.cuda.graph(graph):
        y += 1
        for call in calls:
            with pytest.raises(fm.HIPError):
                call()
        _, n = fm.block_norm_forward(x, pre_weight=w)  # (takes none)
        y += 1
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert (y == 2 * (i + 1)).all()
        assert torch.equal(n, fm.block_norm_forward(x, pre_weight=w)[1])
        again = [call() for call in calls]
        for a, b in zip(eager, again):
            a, b = (t if isinstance(t, tuple) else (t,) for t in (a, b))
            assert all(torch.equal(s, t) for s, t in zip(a, b) if s is not None)
