"""A captured call of the encoder that is lent some of its workspace and not all: it fails, and the graph has nothing of
it.  The memory that it was lent stays as it was."""
import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import _lib, boundary

pytestmark = pytest.mark.gpu


def calls(dtype, device):
    normal = lambda *s: torch.randn(*s, device=device).to(dtype)  # noqa: E731
    out = {}
    # (no whole 16 bytes a head: copies in and out; few rows on many keys, many rows on few: both split)
    for name, sq, sk in (("odd", (1, 40, 2, 30), (1, 50, 1, 30)), ("keys split", (1, 2, 2, 30), (1, 3000, 1, 30)),
                         ("rows split", (1, 1200, 2, 62), (1, 60, 1, 62))):
        q, k, v, do = normal(*sq), normal(*sk), normal(*sk), normal(*sq)
        o, kept = fm.attention_forward(q, k, v, keep=True)
        out[name + ", forward"] = lambda q=q, k=k, v=v: fm.attention_forward(q, k, v, keep=True)[0]
        out[name + ", pullback"] = lambda x=(do, q, k, v, o, kept): fm.attention_pullback(*x)[0]
    q, k, w, table = normal(2, 9, 4, 64), normal(2, 9, 2, 64), normal(64), fm.rotary_table(9, 64, device=device)
    out["rotary"] = lambda: fm.head_rotary_pullback(q, k, q, k, table, q_weight=w, k_weight=w)[0]
    de, ids = normal(400, 136), torch.randint(0, 72, (400,), device=device)
    out["embed"] = lambda: fm.embed_tokens_pullback(de, ids, 70)
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_part_of_the_workspace(dtype, device):
    for name, call in calls(dtype, device).items():
        want = call()
        torch.cuda.synchronize()
        boundary._this_thread()
        for most in range(20):
            lent = []

            def lend(nbytes, stream):
                if len(lent) == most or nbytes > memory.shape[1]:
                    return None
                lent.append(memory[len(lent)][:nbytes])
                return lent[-1].data_ptr()

            memory = torch.full((20, 1 << 22), 0x5a, dtype=torch.uint8, device=device)
            lender = _lib.LENDER(lend)
            _lib.lib().fms_set_workspace_lender(lender)
            try:
                y = torch.zeros(8, device=device)
                graph = torch.cuda.CUDAGraph()
                failed = False
                with torch.cuda.graph(graph):
                    y += 1
                    try:
                        got = call()
                    except fm.HIPError:
                        failed = True
                    y += 1
                for i in range(3):
                    graph.replay()
                    torch.cuda.synchronize()
                    assert (y == 2 * (i + 1)).all()
                    if failed:
                        assert (memory == 0x5a).all(), (name, most)
                    else:
                        assert torch.equal(got, want), (name, most)
                    call()
                    torch.cuda.synchronize()
                    memory.fill_(0x5a)
                    lent.clear()
            finally:
                boundary._this_thread()
            if not failed:
                break
        assert not failed and most > 0, (name, most)
