"""The encoder's operators as they are used: together, in front of MaxSim; captured into graphs and replayed on new
data; on several streams and threads at once."""
import threading

import pytest
import torch

import flashmaxsim as fm
from flashmaxsim import _lib, boundary

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


# ---- a whole encoder layer -----------------------------------------------------------------

H, HK, HEAD, DIM, HIDDEN, EMBED, VOCABULARY = 4, 2, 32, 128, 192, 64, 300


def parameters(device, dtype):
    g = torch.Generator(device=device).manual_seed(0)
    normal = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    matrix = lambda rows, cols: normal(rows, cols) * cols ** -0.5  # noqa: E731
    p = {"table": normal(VOCABULARY, DIM) * 0.1, "qkv": matrix((H + 2 * HK) * HEAD, DIM), "out": matrix(DIM, H * HEAD),
         "wg": matrix(HIDDEN, DIM), "wu": matrix(HIDDEN, DIM), "down": matrix(DIM, HIDDEN), "proj": matrix(EMBED, DIM)}
    p |= {n: 1 + 0.1 * normal(HEAD if n in ("wq", "wk") else DIM) for n in ("n1", "n2", "n3", "wq", "wk")}
    return {n: t.to(dtype).requires_grad_() for n, t in p.items()}


def linear(x, w):
    return (x.flatten(0, 1) @ w.t()).view(*x.shape[:2], -1)


def encode(p, ids):
    """ids (B, T), 0 for padding -> embeddings (B, T, EMBED) by this package."""
    mask = ids > 0
    x = fm.embed_tokens(ids, p["table"], DIM ** 0.5)
    _, n = fm.block_norm(x, pre_weight=p["n1"])
    heads = linear(n, p["qkv"]).view(*ids.shape, H + 2 * HK, HEAD)
    q, k, v = heads.split([H, HK, HK], 2)
    q, k = fm.head_rotary(q, k, fm.rotary_table(ids.shape[1], HEAD, device=ids.device), q_weight=p["wq"],
                          k_weight=p["wk"])
    o = fm.attention(q, k, v, mask, mask, window=9)
    x, n = fm.block_norm(x, linear(o.flatten(2), p["out"]), pre_weight=p["n2"])
    f = linear(fm.gated_ffn(n, p["wg"], p["wu"]), p["down"])
    _, n = fm.block_norm(x, f, pre_weight=p["n3"])
    return linear(n, p["proj"])


def encode_plain(p, ids):
    """The same from elementary operations."""
    norm = lambda a, w: a * (a.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
    B, T = ids.shape
    real = ids > 0
    x = torch.where(real[..., None], p["table"][(ids - 1).clamp(min=0).long()] * DIM ** 0.5, 0.0)
    heads = (norm(x, p["n1"]) @ p["qkv"].t()).view(B, T, H + 2 * HK, HEAD)
    q, k, v = heads.split([H, HK, HK], 2)
    t = fm.rotary_table(T, HEAD, device=ids.device).to(x.dtype)[:, None]
    cos, sin = t.split(HEAD // 2, -1)

    def turn(y):
        a, b = y.split(HEAD // 2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q, k = turn(norm(q, p["wq"])), turn(norm(k, p["wk"]))
    k, v = k.repeat_interleave(H // HK, 2), v.repeat_interleave(H // HK, 2)
    s = (q[:, :, None] * k[:, None]).sum(-1) * HEAD ** -0.5  # (B, Tq, Tk, heads)
    near = (torch.arange(T, device=ids.device)[:, None] - torch.arange(T, device=ids.device)).abs() <= 9
    keep = (near & real[:, :, None] & real[:, None])[..., None]
    s = torch.where(keep, s, -1e30)
    w = torch.softmax(s, 2) * keep
    o = (w[..., None] * v[:, None]).sum(2).flatten(2)
    x = x + o @ p["out"].t()
    n = norm(x, p["n2"])
    x = x + (torch.nn.functional.silu(n @ p["wg"].t()) * (n @ p["wu"].t())) @ p["down"].t()
    return norm(x, p["n3"]) @ p["proj"].t()


def token_ids(device):
    g = torch.Generator(device=device).manual_seed(1)
    q = torch.randint(1, VOCABULARY + 1, (5, 8), generator=g, device=device)
    d = torch.randint(1, VOCABULARY + 1, (5, 31), generator=g, device=device)
    d[1, 20:], d[3, 1:], q[2, 6:] = 0, 0, 0
    return q.int(), d


def test_encoder_layer(device):
    """Embeddings, MaxSim scores and the gradients of every parameter, fp32 against 64 bits.

    Each entry passes a dozen sums of at most 192 terms (a relative 192 * 2^-24 each at worst), norms and a
    softmax that amplify a relative error a few times over: 12 * 192 * 2^-24 * 30 bounds them."""
    far = 12 * 192 * 2.0 ** -24 * 30
    q, d = token_ids(device)
    p = parameters(device, torch.float32)
    wide = {n: t.detach().double().requires_grad_() for n, t in p.items()}
    eq, ed = encode(p, q), encode(p, d)
    wq, wd = encode_plain(wide, q), encode_plain(wide, d)
    for a, b in ((eq, wq), (ed, wd)):
        assert float(((a - b).norm() / b.norm()).detach()) < far
    scores = fm.maxsim(eq, ed, q > 0, d > 0, fm.InBatch())
    sims = torch.einsum("qid,cjd->qcij", wq, wd)
    sims = torch.where((d > 0)[None, :, None], sims, -1e30).amax(-1)
    want = (sims * (q > 0)[:, None]).sum(-1)
    assert float(((scores - want).abs().max() / want.abs().max()).detach()) < far
    target = torch.arange(5, device=device)
    torch.nn.functional.cross_entropy(scores / 20, target).backward()
    torch.nn.functional.cross_entropy(want / 20, target).backward()
    for n, t in p.items():
        g, w = t.grad.double(), wide[n].grad
        assert float((g - w).norm() / w.norm()) < far, n


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_encoder_layer_in_16_bits(dtype, device):
    """The chain runs, padding stays out of it, and its embeddings are as far from 64 bits as a dozen roundings
    of states of like size take them (each at most half a step, amplified a few times over)."""
    q, d = token_ids(device)
    p = parameters(device, dtype)
    wide = {n: t.detach().double() for n, t in p.items()}
    ed = encode(p, d)
    want = encode_plain(wide, d)
    assert float((ed - want).norm() / want.norm()) < 12 * torch.finfo(dtype).eps / 2 * 3
    fm.maxsim(encode(p, q), ed, q > 0, d > 0, fm.InBatch()).diagonal().sum().backward()
    for n, t in p.items():
        assert torch.isfinite(t.grad).all() and t.grad.any(), n
    unseen = torch.ones(VOCABULARY, dtype=torch.bool, device=device)
    unseen[torch.cat([q.flatten(), d.flatten()]).long().unique()[1:] - 1] = False
    assert not p["table"].grad[unseen].any()


# ---- graphs ----------------------------------------------------------------------------------

def cases(dtype, device):
    """{name: (inputs to change, call)}: every kernel and path that takes workspace."""
    g = torch.Generator(device=device).manual_seed(2)
    normal = lambda *s: torch.randn(*s, generator=g, device=device).to(dtype)  # noqa: E731
    out = {}

    def attend(name, sq, sk, **args):
        q, k, v, do = normal(*sq), normal(*sk), normal(*sk), normal(*sq)

        def call():
            o, kept = fm.attention_forward(q, k, v, keep=True, **args)
            return (o, *fm.attention_pullback(do, q, k, v, o, kept, **args))
        out[name] = ([q, k, v, do], call)

    mask = torch.arange(150, device=device)[None] < torch.tensor([[70], [150]], device=device)
    cu = torch.tensor([1, 40, 40, 131], dtype=torch.int32, device=device)
    attend("masked", (2, 150, 4, 64), (2, 150, 2, 64), qmask=mask, kmask=mask, causal=True)
    attend("odd", (1, 40, 2, 30), (1, 50, 1, 30))
    attend("keys split", (1, 2, 2, 128), (1, 3000, 1, 128))
    attend("rows split", (1, 1200, 2, 64), (1, 60, 1, 64))
    attend("ragged", (135, 2, 64), (135, 2, 64), cu_q=cu, cu_k=cu, max_q=91, max_k=91, window=20)
    q, k, dq, dk, w = normal(2, 9, 4, 64), normal(2, 9, 2, 64), normal(2, 9, 4, 64), normal(2, 9, 2, 64), normal(64)
    table = fm.rotary_table(9, 64, device=device)

    def turn():
        y = fm.head_rotary_forward(q, k, table, q_weight=w, k_weight=w)
        return (*y, *fm.head_rotary_pullback(dq, dk, q, k, table, q_weight=w, k_weight=w))
    out["rotary"] = ([q, k, dq, dk, w], turn)
    weight, de = normal(70, 136), normal(400, 136)
    ids = torch.randint(0, 72, (400,), generator=g, device=device)
    ids[::3] = 5

    def look_up():
        return fm.embed_tokens_forward(ids, weight, 2.0), fm.embed_tokens_pullback(de, ids, 70, 2.0)
    out["embed"] = ([weight, de], look_up)
    return out


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_and_replayed(dtype, device):
    """Each replay, on new data, with other calls between them, gives what an eager call gives, bit for bit."""
    for name, (inputs, call) in cases(dtype, device).items():
        call()  # (loads the kernels)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for i in range(4):
            for t in inputs:
                t.copy_(torch.randn(t.shape, generator=torch.Generator(device=device).manual_seed(i), device=device)
                        * 10.0 ** (i - 2))
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (name, i)


def test_two_graphs_share_no_workspace(device):
    """Two captured calls, replayed in turn on two streams at once."""
    made = []
    for seed in range(2):
        inputs, call = cases(torch.float16, device)["keys split"]
        for t in inputs:
            t.mul_(seed + 1)
        want = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        made.append((graph, got, want, inputs))
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(3):
        for (graph, *_), s in zip(made, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, got, want, _ in made:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["masked", "odd", "keys split", "rows split", "rotary", "embed"])
def test_captured_without_workspace_fails(name, device):
    """A captured call that needs workspace and is lent none fails and adds nothing to the graph."""
    inputs, call = cases(torch.float16, device)[name]
    want = call()
    torch.cuda.synchronize()
    boundary._this_thread()
    _lib.lib().fms_set_workspace_lender(_lib.LENDER(0))
    try:
        y = torch.zeros(8, device=device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y += 1
            with pytest.raises(fm.HIPError):
                call()
            y += 1
        for i in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert (y == 2 * (i + 1)).all()
            assert all(torch.equal(a, b) for a, b in zip(call(), want))  # from the pool
    finally:
        boundary._this_thread()


# ---- streams and threads ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_streams_and_threads(dtype, device):
    """Calls of several threads, each on its own stream, at once."""
    made = cases(dtype, device)
    want = {name: call() for name, (_, call) in made.items()}
    torch.cuda.synchronize()
    bad = []

    def work(names):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    for name in names:
                        got = made[name][1]()
                        stream.synchronize()
                        if not all(torch.equal(a, b) for a, b in zip(got, want[name])):
                            bad.append(name)
        except Exception as e:  # noqa: BLE001
            bad.append(repr(e))

    names = list(made)
    threads = [threading.Thread(target=work, args=(names[i:] + names[:i],)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
