"""More operators of the encoder before MaxSim, whose speed is tracked: attention over heads, the
norm and rotation of its queries and keys, and the lookup of token embeddings.

With the token block's operators they turn token ids into the embeddings that MaxSim scores.  Each
case below is one pass: forward only (indexing, search) or forward and pullback (training).
``run`` computes the operators from elementary torch operations in 32 bits, or, with ``own`` set,
calls this repository's entry points on the same inputs.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6


def _framework():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashmaxsim.jl_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flashmaxsim
    return flashmaxsim


# ---- cases -----------------------------------------------------------------------------

def _attention(name, seqs, queries, keys, heads, kv_heads, dim, dtype, train, lengths="full",
               causal=False, window=0):
    """lengths: "full" (all keys count), "mask" (padded, masks of both sides) or "ragged" (token
    rows of all sequences behind one another; as many queries as keys).  window 0: none."""
    return {"name": name, "op": "attention", "seqs": seqs, "queries": queries, "keys": keys,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "train": train,
            "lengths": lengths, "causal": causal, "window": window}


def _rotary(name, seqs, tokens, heads, kv_heads, dim, turned, dtype, kind, pairing, placed, train):
    """turned: how many of a head's values the rotation takes; placed: positions are given."""
    return {"name": name, "op": "rotary", "seqs": seqs, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "turned": turned, "dtype": dtype, "kind": kind,
            "pairing": pairing, "placed": placed, "train": train}


def _embed(name, seqs, tokens, vocabulary, dim, dtype, train):
    return {"name": name, "op": "embed", "seqs": seqs, "tokens": tokens, "vocabulary": vocabulary,
            "dim": dim, "dtype": dtype, "train": train}


def listed():
    return [
        # one query's 32 tokens among themselves, at search time: all latency
        _attention("attention_query", 1, 32, 32, 12, 12, 64, "f16", False),
        # a single token that gathers a long page, heads in groups of four
        _attention("attention_one_token", 1, 1, 32768, 16, 4, 128, "bf16", False),
        # 256 padded documents of up to 180 tokens, at indexing time
        _attention("attention_documents", 256, 180, 180, 12, 12, 64, "bf16", False, "mask"),
        # a training step's documents: forward, then the gradients of queries, keys and values
        _attention("attention_train", 128, 180, 180, 16, 16, 64, "bf16", True, "mask"),
        # documents of very different lengths behind one another, each token seeing its neighbours
        _attention("attention_train_ragged", 48, 1999, 1999, 12, 12, 64, "f16", True, "ragged", False, 64),
        # one long page under a causal mask, heads in groups of four
        _attention("attention_train_long", 1, 8192, 8192, 16, 4, 128, "bf16", True, "full", True),
        # training in 32 bits, odd lengths, a head width that is no whole tile
        _attention("attention_train_f32", 16, 237, 301, 6, 6, 48, "f32", True, "mask"),
        # norm and rotation of one query's heads
        _rotary("rotary_query", 1, 32, 12, 12, 64, 64, "f16", "rms", "halves", False, False),
        # the same in training, on slices of one projection's output
        _rotary("rotary_train", 128, 180, 16, 16, 64, 64, "bf16", "rms", "halves", False, True),
        # 32 bits, few key heads, part of an odd-sized head turned, neighbours paired, positions given
        _rotary("rotary_train_odd", 27, 37, 9, 3, 50, 36, "f32", "layer", "neighbours", True, True),
        # the ids of one query looked up
        _embed("embed_query", 1, 32, 32768, 768, "f16", False),
        # a training step's documents: lookup, then the gradient of the whole table
        _embed("embed_train", 128, 180, 32768, 1024, "bf16", True),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rotary", "embed"])
    dtype, train = rng.choice(["f32", "f16", "bf16", "bf16"]), rng.random() < 0.5
    heads, group = _log(rng, 1, 16), rng.choice([1, 1, 2, 4])
    dim = rng.choice([32, 64, 64, 128, 2 * _log(rng, 8, 64), _log(rng, 16, 128)])
    if op == "attention":
        lengths = rng.choice(["full", "mask", "ragged"])
        keys = _log(rng, 1, 4096)
        queries = keys if lengths == "ragged" or rng.random() < 0.6 else _log(rng, 1, 4096)
        most = (6e7 if dtype == "f32" else 2.5e8) / (queries * keys * heads * group)
        c = _attention("", _log(rng, 1, max(1, min(128, int(most)))), queries, keys, heads * group,
                       heads, dim, dtype, train, lengths, rng.random() < 0.4,
                       rng.choice([0, 0, _log(rng, 1, 512)]))
    elif op == "rotary":
        dim += dim & 1
        turned = dim if rng.random() < 0.6 else 2 * _log(rng, 1, dim // 2)
        c = _rotary("", _log(rng, 1, 128), _log(rng, 1, 180), heads, max(1, heads // group), dim,
                    turned, dtype, rng.choice(["rms", "layer", "none"]),
                    rng.choice(["halves", "neighbours"]), rng.random() < 0.5, train)
    else:
        c = _embed("", _log(rng, 1, 128), _log(rng, 1, 180), _log(rng, 64, 32768),
                   rng.choice([_log(rng, 16, 1024), 32 * _log(rng, 1, 32)]), dtype, train)
    del c["name"]
    return c


def _lengths(c):
    """How many tokens each sequence has: the first all, the others falling off unevenly."""
    i = np.arange(c["seqs"])
    share = np.where(i == 0, 1.0, ((i * 0.6180339887498949) % 1.0) ** 1.5)
    both = [np.maximum(1, np.round(share * c[k])).astype(np.int64) for k in ("queries", "keys")]
    return [np.full_like(n, n[0]) for n in both] if c["lengths"] == "full" else both


def _pairs(c):
    """(query, key) pairs that count, of one head."""
    total = 0
    for nq, nk in zip(*_lengths(c)):
        # (padded sequences keep their place in the padded shape)
        shift = c["keys"] - c["queries"] if c["lengths"] == "mask" else nk - nq
        i = np.arange(nq) + shift
        first = np.maximum(0, i - c["window"]) if c["window"] else np.zeros_like(i)
        last = np.full_like(i, nk - 1)
        if c["window"]:
            last = np.minimum(last, i + c["window"])
        if c["causal"]:
            last = np.minimum(last, i)
        total += int(np.maximum(0, last - first + 1).sum())
    return total


def work(case):
    c, e = case, 4 if case["dtype"] == "f32" else 2
    if c["op"] == "attention":
        nq, nk = (int(n.sum()) for n in _lengths(c))
        n = 2 * nq * c["heads"] + 2 * nk * c["kv_heads"]  # q and o, k and v
        # two products forward; five more for the gradients, and their cotangent and three results
        n += (2 * nq * c["heads"] + 2 * nk * c["kv_heads"]) if c["train"] else 0
        return {"bytes": e * c["dim"] * n,
                "flops": 2 * c["dim"] * c["heads"] * _pairs(c) * (7 if c["train"] else 2)}
    if c["op"] == "rotary":
        n = c["seqs"] * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        # in and out; in training the cotangents in and the gradients out as well
        return {"bytes": e * n * (4 if c["train"] else 2), "flops": n * (40 if c["train"] else 15)}
    n = c["seqs"] * c["tokens"]
    nbytes = 4 * n + e * (min(n, c["vocabulary"]) + n) * c["dim"]
    if c["train"]:
        nbytes += e * (n + c["vocabulary"]) * c["dim"]
    return {"bytes": nbytes, "flops": n * c["dim"] * (2 if c["train"] else 1)}


# ---- inputs ----------------------------------------------------------------------------

def _inputs(case, seed):
    c, dt = case, _TYPES[case["dtype"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dt)

    if c["op"] == "attention":
        b, tq, tk, h, hk, d = (c[k] for k in ("seqs", "queries", "keys", "heads", "kv_heads", "dim"))
        nq, nk = _lengths(c)
        s = {"cu": None, "qmask": None, "kmask": None}
        if c["lengths"] == "ragged":  # 1-based first rows, and one past the last
            s["cu"] = torch.from_numpy(np.concatenate([[1], 1 + np.cumsum(nk)]).astype(np.int32)).cuda()
            lead_q = lead_k = (int(nk.sum()),)
        else:
            lead_q, lead_k = (b, tq), (b, tk)
        if c["lengths"] == "mask":
            s["qmask"], s["kmask"] = (torch.arange(t, device="cuda") < torch.from_numpy(n).cuda()[:, None]
                                      for t, n in ((tq, nq), (tk, nk)))
        # queries and keys after their norm and rotation; values a slice of the projection's output
        s["q"], s["k"] = normal(*lead_q, h, d), normal(*lead_k, hk, d)
        s["v"] = normal(*lead_k, h + 2 * hk, d).narrow(-2, h + hk, hk)
        if c["train"]:
            s["do"] = normal(*lead_q, h, d, scale=0.05)
        return s
    if c["op"] == "rotary":
        b, t, h, hk, d, r = (c[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "turned"))
        qkv = normal(b, t, h + 2 * hk, d, scale=1.5, shift=0.1)
        rows = t + 75 if c["placed"] else t
        angle = (torch.arange(rows, dtype=torch.float64, device="cuda")[:, None]
                 * 10000.0 ** (torch.arange(r // 2, dtype=torch.float64, device="cuda") * (-2.0 / r)))
        s = {"q": qkv.narrow(2, 0, h), "k": qkv.narrow(2, h, hk), "wq": None, "wk": None,
             "positions": None, "table": torch.cat([angle.cos(), angle.sin()], 1).float()}
        if c["placed"]:  # 1-based rows of the table
            first = torch.randint(1, 76, (b, 1), generator=g, device="cuda")
            s["positions"] = (first + torch.arange(t, device="cuda")).int()
        if c["kind"] != "none":
            s["wq"], s["wk"] = normal(d, scale=0.1, shift=1.0), normal(d, scale=0.1, shift=1.0)
        if c["train"]:
            s["dq"], s["dk"] = normal(b, t, h, d, scale=0.05), normal(b, t, hk, d, scale=0.05)
        return s
    b, t, v, d = (c[k] for k in ("seqs", "tokens", "vocabulary", "dim"))
    # the n-th frequent token about 1 / n of the time, frequent ones anywhere in the table; id 0 pads
    rank = (v ** torch.rand(b, t, generator=g, device="cuda", dtype=torch.float64)).long().clamp(1, v)
    ids = torch.randperm(v, generator=g, device="cuda")[rank - 1] + 1
    left = torch.rand(b, 1, generator=g, device="cuda") * 0.6 * t
    ids = torch.where(torch.arange(t, device="cuda") < t - left, ids, 0).int()
    s = {"ids": ids, "weight": normal(v, d, scale=0.02)}
    if c["train"]:
        s["de"] = normal(b, t, d, scale=0.05)
    return s


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ---- plain forms -----------------------------------------------------------------------

def _padded(s, t, length):
    """Ragged rows (tokens, heads, dim) as (sequences, length, heads, dim), and which rows are real."""
    first = s["cu"].long() - 1
    at = first[:-1, None] + torch.arange(length, device=t.device)
    real = at < first[1:, None]
    return t[torch.where(real, at, 0)], real


def _counting(c, nq, nk, tq, tk):
    """Which (query, key) pairs count by their positions: (sequences or 1, tq, tk), or None."""
    if not c["causal"] and not c["window"]:
        return None
    away = (torch.arange(tk, device="cuda") - torch.arange(tq, device="cuda")[:, None]
            - (nk - nq)[:, None, None])
    counts = away <= (0 if c["causal"] else tk + tq)
    return counts & (away.abs() <= c["window"]) if c["window"] else counts


def _plain_attention(s):
    c, dt = s["case"], s["q"].dtype
    b, tq, tk, h, hk, d = (c[k] for k in ("seqs", "queries", "keys", "heads", "kv_heads", "dim"))
    q, k, v, do = (None if t is None else t.float() for t in (s["q"], s["k"], s["v"], s.get("do")))
    qreal, kreal = s["qmask"], s["kmask"]
    nq, nk = (torch.full((1,), t, device="cuda") for t in (tq, tk))
    if s["cu"] is not None:
        (q, qreal), (k, kreal), (v, _) = _padded(s, q, tq), _padded(s, k, tk), _padded(s, v, tk)
        do = None if do is None else _padded(s, do, tq)[0]
        nq = nk = (s["cu"][1:] - s["cu"][:-1]).long()

    def by_head(t):  # (sequences, key heads, queries of the group, dim) and the like
        n = t.shape[1]
        t = t.view(b, n, hk, -1, d).permute(0, 2, 3, 1, 4)
        return t.reshape(b, hk, -1, d)

    def back(t, n):
        return t.view(b, hk, -1, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, -1, d).to(dt)

    keep = _counting(c, nq, nk, tq, tk)
    if qreal is not None:
        real = qreal[:, :, None] & kreal[:, None, :]
        keep = real if keep is None else keep & real
        # (what a mask leaves out may hold anything)
        q = torch.where(qreal[:, :, None, None], q, 0)
        k, v = (torch.where(kreal[:, :, None, None], t, 0) for t in (k, v))
        do = None if do is None else torch.where(qreal[:, :, None, None], do, 0)
    scale = d ** -0.5
    q, k, v = by_head(q), by_head(k), by_head(v)
    p = (q @ k.transpose(2, 3)).mul_(scale).view(b, hk, h // hk, tq, tk)
    if keep is not None:
        keep = keep[:, None, None]
        p.masked_fill_(~keep, -math.inf)
        top = p.amax(-1, keepdim=True)
        p.sub_(torch.where(top == -math.inf, 0, top)).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(torch.where(total == 0, 1, total))
    else:
        p.sub_(p.amax(-1, keepdim=True)).exp_()
        p.div_(p.sum(-1, keepdim=True))
    p = p.view(b, hk, -1, tk)
    o = p @ v
    if not c["train"]:
        out = {"o": back(o, tq)}
    else:
        do = by_head(do)
        ds = do @ v.transpose(2, 3)
        delta = (ds * p).sum(-1, keepdim=True)
        ds.sub_(delta).mul_(p)
        out = {"o": back(o, tq), "dq": back(ds @ k * scale, tq),
               "dk": back(ds.transpose(2, 3) @ q * scale, tk), "dv": back(p.transpose(2, 3) @ do, tk)}
    if s["cu"] is not None:
        out = {name: t[qreal] for name, t in out.items()}
    return out


def _standard(a, kind):
    """a without its mean (layer) over its spread, and 1 / spread, row by row."""
    if kind == "layer":
        a = a - a.mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((a * a).mean(-1, keepdim=True) + _EPS)
    return a * inv, inv


def _turn(t, cos, sin, r, pairing):
    """The first r values of t's heads turned, in pairs (i, i + r / 2) or (2 i, 2 i + 1)."""
    head = t[..., :r]
    if pairing == "halves":
        a, b = head[..., :r // 2], head[..., r // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, t[..., r:]], -1)


def _plain_rotary(s):
    c, dt = s["case"], s["q"].dtype
    r, kind = c["turned"], c["kind"]
    rows = (s["table"][:c["tokens"]] if s["positions"] is None else s["table"][s["positions"].long() - 1])
    cos, sin = rows[..., None, :r // 2], rows[..., None, r // 2:]
    out = {}
    for name in ("q", "k"):
        x, w = s[name].float(), s["w" + name]
        hat, inv = x, None
        if w is not None:
            hat, inv = _standard(x, kind)
            x = hat * w.float()
        out[name] = _turn(x, cos, sin, r, c["pairing"]).to(dt)
        if c["train"]:
            d = _turn(s["d" + name].float(), cos, -sin, r, c["pairing"])
            if w is not None:
                out["dw" + name] = (d * hat).sum((0, 1, 2)).to(dt)
                d = d * w.float()
                d = d - hat * (d * hat).mean(-1, keepdim=True)
                d = (d - d.mean(-1, keepdim=True) if kind == "layer" else d) * inv
            out["d" + name] = d.to(dt)
    return out


_SCALE = 27.7  # of looked-up rows: about the root of their width, as encoders have it


def _plain_embed(s):
    c, dt = s["case"], s["weight"].dtype
    ids = s["ids"].long()
    real = ids > 0
    rows = s["weight"][(ids - 1).clamp(min=0)].float() * _SCALE
    out = {"e": torch.where(real[..., None], rows, 0).to(dt)}
    if c["train"]:
        total = torch.zeros(c["vocabulary"] + 1, c["dim"], device="cuda")
        total.index_add_(0, ids.view(-1), s["de"].float().view(-1, c["dim"]))
        out["dweight"] = (total[1:] * _SCALE).to(dt)
    return out


# ---- the framework's operators ---------------------------------------------------------

def _own_attention(s):
    fm, c = _framework(), s["case"]
    args = dict(causal=c["causal"], window=c["window"] or None)
    if s["cu"] is not None:
        args |= dict(cu_q=s["cu"], cu_k=s["cu"], max_q=c["queries"], max_k=c["keys"])
    else:
        args |= dict(qmask=s["qmask"], kmask=s["kmask"])
    if not c["train"]:
        return {"o": fm.attention_forward(s["q"], s["k"], s["v"], **args)}
    o, kept = fm.attention_forward(s["q"], s["k"], s["v"], keep=True, **args)
    dq, dk, dv = fm.attention_pullback(s["do"], s["q"], s["k"], s["v"], o, kept, **args)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _own_rotary(s):
    fm, c = _framework(), s["case"]
    args = dict(positions=s["positions"], q_weight=s["wq"], k_weight=s["wk"], pairing=c["pairing"],
                kind="rms" if c["kind"] == "none" else c["kind"], eps=_EPS)
    q, k = fm.head_rotary_forward(s["q"], s["k"], s["table"], **args)
    out = {"q": q, "k": k}
    if c["train"]:
        dq, dk, dwq, dwk = fm.head_rotary_pullback(s["dq"], s["dk"], s["q"], s["k"], s["table"], **args)
        out |= {"dq": dq, "dwq": dwq, "dk": dk, "dwk": dwk}
    names = ("q", "dwq", "dq", "k", "dwk", "dk")  # the plain form's order
    return {n: out[n] for n in names if out.get(n) is not None}


def _own_embed(s):
    fm, c = _framework(), s["case"]
    out = {"e": fm.embed_tokens_forward(s["ids"], s["weight"], _SCALE)}
    if c["train"]:
        out["dweight"] = fm.embed_tokens_pullback(s["de"], s["ids"], c["vocabulary"], _SCALE)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "rotary": _own_rotary, "embed": _own_embed}[op](state)
    return {"attention": _plain_attention, "rotary": _plain_rotary, "embed": _plain_embed}[op](state)


# ---- 64 bits ---------------------------------------------------------------------------

def _exact_attention(s, c):
    b, tq, tk, h, hk, d = (c[k] for k in ("seqs", "queries", "keys", "heads", "kv_heads", "dim"))
    dev, real_q, real_k = "cuda", s["qmask"], s["kmask"]
    place = None
    if s["cu"] is not None:  # where each sequence's rows lie in the padded shape
        n = (s["cu"][1:] - s["cu"][:-1]).long()
        place = torch.arange(tq, device=dev) < n[:, None]
        real_q = real_k = place
    lengths = [n if place is not None else torch.full((b,), t, device=dev) for t in (tq, tk)]

    def wide(t, real, length):
        """Double, padded, zero where masked."""
        if place is not None:
            out = torch.zeros(b, length, *t.shape[1:], dtype=torch.float64, device=dev)
            out[place] = t.double()
            return out
        t = t.double()
        return t if real is None else torch.where(real[..., None, None], t, 0.0)

    q, k, v = wide(s["q"], real_q, tq), wide(s["k"], real_k, tk), wide(s["v"], real_k, tk)
    do = wide(s["do"], real_q, tq) if c["train"] else None
    i = torch.arange(tq, device=dev)[None, :, None] + (lengths[1] - lengths[0])[:, None, None]
    j = torch.arange(tk, device=dev)[None, None, :]
    out_of = torch.zeros(b, tq, tk, dtype=torch.bool, device=dev)
    if c["causal"]:
        out_of |= j > i
    if c["window"]:
        out_of |= (j - i > c["window"]) | (i - j > c["window"])
    if real_q is not None:
        out_of |= ~real_q[:, :, None]
        out_of |= ~real_k[:, None, :]
    empty = out_of.all(-1)
    results = {name: torch.zeros_like(t) for name, t in
               (("o", q), ("dq", q), ("dk", k), ("dv", v)) if name == "o" or c["train"]}
    for head in range(h):
        kv = head // (h // hk)
        x = [t[:, :, n].contiguous().requires_grad_(c["train"]) for t, n in ((q, head), (k, kv), (v, kv))]
        score = torch.bmm(x[0], x[1].transpose(1, 2)) / math.sqrt(d)
        score = score.masked_fill(out_of & ~empty[..., None], -math.inf)
        y = torch.bmm(torch.softmax(score, -1), x[2]).masked_fill(empty[..., None], 0.0)
        results["o"][:, :, head] = y.detach()
        if c["train"]:
            gq, gk, gv = torch.autograd.grad(y, x, do[:, :, head].contiguous())
            results["dq"][:, :, head] = gq
            results["dk"][:, :, kv] += gk
            results["dv"][:, :, kv] += gv
    return {name: t if place is None else t[place] for name, t in results.items()}


def exact(case, seed):
    """The definitions in 64 bits, gradients by differentiating the definition."""
    s, c = _inputs(case, seed), case
    if c["op"] == "attention":
        return _exact_attention(s, c)
    if c["op"] == "rotary":
        r, half = c["turned"], c["turned"] // 2
        at = (torch.arange(c["tokens"], device="cuda")[None] if s["positions"] is None
              else s["positions"].long() - 1)
        table = s["table"].double()[at]
        phase = torch.complex(table[..., :half], table[..., half:])[:, :, None]
        out = {}
        for name in ("q", "k"):
            v = [s[name].double().requires_grad_(c["train"])]
            y = v[0]
            if s["w" + name] is not None:
                v.append(s["w" + name].double().requires_grad_(c["train"]))
                if c["kind"] == "layer":
                    y = y - y.mean(-1, keepdim=True)
                y = y * (y.pow(2).sum(-1, keepdim=True) / c["dim"] + _EPS).rsqrt() * v[1]
            head, rest = y[..., :r], y[..., r:]
            shape = (2, half) if c["pairing"] == "halves" else (half, 2)
            pair = head.unflatten(-1, shape)
            pair = pair if c["pairing"] == "neighbours" else pair.transpose(-1, -2)
            turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * phase)
            turned = turned if c["pairing"] == "neighbours" else turned.transpose(-1, -2)
            y = torch.cat([turned.flatten(-2), rest], -1)
            out[name] = y.detach()
            if c["train"]:
                grads = torch.autograd.grad(y, v, s["d" + name].double())
                if len(grads) == 2:
                    out["dw" + name] = grads[1]
                out["d" + name] = grads[0]
        return out
    w = torch.cat([torch.zeros(1, c["dim"], dtype=torch.float64, device="cuda"), s["weight"].double()])
    ids = s["ids"].long()
    out = {"e": w.index_select(0, ids.flatten()).view(*ids.shape, -1) * _SCALE}
    if c["train"]:  # sums of sorted runs, as differences of running sums
        order = ids.flatten().argsort(stable=True)
        run = s["de"].double().view(-1, c["dim"])[order].cumsum(0)
        run = torch.cat([torch.zeros_like(run[:1]), run])
        ends = torch.bincount(ids.flatten(), minlength=c["vocabulary"] + 1).cumsum(0)
        out["dweight"] = (run[ends[1:]] - run[ends[:-1]]) * _SCALE
    return out
