"""The token-block operators whose speed is tracked: gated feed-forward, block norms, AdamW.

A token block turns an encoder's token states into the embeddings that MaxSim scores, and an
optimiser step uses MaxSim's gradients to train it.  Each case below is one pass through one of
the three operators that do this: forward only (serving), forward and pullback (training), or one
step over a list of parameters.  ``run`` computes the operators from elementary torch operations
in 32 bits, or, with ``own`` set, calls this repository's entry points on the same inputs.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BLOCK = 256  # elements of a parameter that share the scale of their 8-bit moments
_BETAS, _EPS, _DECAY, _LR = (0.9, 0.999), 1e-8, 1e-2, 1e-3


def _framework():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashmaxsim.jl_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flashmaxsim
    return flashmaxsim


# ---- cases -----------------------------------------------------------------------------

def _ffn(name, tokens, dim, hidden, dtype, act, train):
    return {"name": name, "op": "ffn", "tokens": tokens, "dim": dim, "hidden": hidden,
            "dtype": dtype, "act": act, "train": train}


def _norm(name, seqs, tokens, dim, dtype, kind, form, gate, train):
    return {"name": name, "op": "norm", "seqs": seqs, "tokens": tokens, "dim": dim,
            "dtype": dtype, "kind": kind, "form": form, "gate": gate, "train": train}


def _adamw(name, tensors, elements, dtype, bits, master):
    return {"name": name, "op": "adamw", "tensors": tensors, "elements": elements,
            "dtype": dtype, "bits": bits, "master": master}


def listed():
    return [
        # one token through a wide block: all latency and weight bytes
        _ffn("ffn_one_token", 1, 1024, 4096, "bf16", "silu", False),
        # the 32 tokens of one query, at search time
        _ffn("ffn_query", 32, 768, 2048, "f16", "gelu", False),
        # 256 documents of 180 tokens, at indexing time
        _ffn("ffn_documents", 256 * 180, 768, 2048, "bf16", "gelu_tanh", False),
        # a training step's documents: forward, then the gradients of states and weights
        _ffn("ffn_train", 128 * 180, 1024, 4096, "bf16", "silu", True),
        # a small batch of odd lengths through a block whose rows are no whole 16-byte units
        _ffn("ffn_train_odd", 1237, 200, 531, "f16", "gelu", True),
        # training in 32 bits throughout
        _ffn("ffn_train_f32", 4096, 384, 1024, "f32", "silu", True),
        # the norm before a block, one query
        _norm("norm_query", 1, 32, 768, "f16", "rms", "pre", "none", False),
        # end of one block and start of the next, indexing, one gate vector for all tokens
        _norm("norm_documents", 256, 180, 768, "bf16", "layer", "both", "shared", False),
        # the same in training, a gate for each document
        _norm("norm_train", 128, 180, 1024, "bf16", "rms", "both", "sequence", True),
        # odd width, 32 bits, no norm of the branch
        _norm("norm_train_odd", 27, 37, 531, "f32", "layer", "plain", "sequence", True),
        # an encoder's worth of small and middling tensors, 16-bit weights over 32-bit masters
        _adamw("adamw_many", 148, 8_000_001, "bf16", 32, True),
        # few large tensors with the moments in 8 bits
        _adamw("adamw_8bit", 12, 64_000_000, "bf16", 8, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly whole 16-byte units, else anything."""
    n = _log(rng, lo, hi)
    n = n if rng.random() < 0.4 else max(lo, n // 32 * 32)
    return n + 32 if n == 3072 else n


def draw(rng):
    op = rng.choice(["ffn", "ffn", "norm", "norm", "adamw"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "ffn":
        train = rng.random() < 0.5
        dim, hidden = _width(rng, 64, 1024), _width(rng, 128, 4096)
        most = (2.5e11 if dtype != "f32" else 1.2e10) / (dim * hidden) / (3 if train else 1)
        tokens = _log(rng, 1, max(2, min(46080, most)))
        c = _ffn("", tokens + (tokens == 3072), dim, hidden, dtype,
                 rng.choice(["silu", "gelu", "gelu_tanh"]), train)
    elif op == "norm":
        c = _norm("", _log(rng, 1, 256), _log(rng, 1, 180), _width(rng, 64, 1024), dtype,
                  rng.choice(["rms", "layer"]), rng.choice(["pre", "post", "plain", "both"]),
                  rng.choice(["none", "shared", "sequence"]), rng.random() < 0.5)
    else:
        tensors = _log(rng, 1, 200)
        c = _adamw("", tensors, max(tensors, _log(rng, 1000, 32_000_000)), dtype,
                   rng.choice([8, 32]), dtype != "f32" and rng.random() < 0.5)
    del c["name"]
    return c


def _sizes(c):
    """The parameters' element counts: shares that fall off, as a model's matrices and vectors do."""
    k, n = c["tensors"], c["elements"]
    shares = [1.0 / (1 + i % 7) ** 3 for i in range(k)]
    sizes = [max(1, int(n * s / sum(shares))) for s in shares]
    sizes[0] += max(0, n - sum(sizes))
    return sizes


def work(case):
    c, e = case, 4 if case["dtype"] == "f32" else 2
    if c["op"] == "ffn":
        t, k, f = c["tokens"], c["dim"], c["hidden"]
        nbytes, flops = e * (t * k + 2 * f * k + t * f), 4 * t * k * f
        if c["train"]:
            nbytes, flops = nbytes + e * (t * f + t * k + 2 * f * k), 3 * flops
        return {"bytes": nbytes, "flops": flops}
    if c["op"] == "norm":
        rows, d = c["seqs"] * c["tokens"], c["dim"]
        n = {"pre": 2, "post": 3, "plain": 4, "both": 4}[c["form"]]
        if c["train"]:  # and dr / dn in, dx / df out
            n += {"pre": 2, "post": 3, "plain": 4, "both": 4}[c["form"]]
        return {"bytes": e * rows * d * n, "flops": 20 * rows * d}
    per = 2 * e  # gradient read, parameter written
    per += 8 if c["master"] else e
    # moments: 32 bits read and written; 8 bits read, written, and their values given back
    per += 16 if c["bits"] == 32 else 4 + 8
    return {"bytes": per * sum(_sizes(c)), "flops": 20 * sum(_sizes(c))}


# ---- inputs ----------------------------------------------------------------------------

def _inputs(case, seed):
    c, dt = case, _TYPES[case["dtype"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    if c["op"] == "ffn":
        t, k, f = c["tokens"], c["dim"], c["hidden"]
        s = {"x": normal(t, k), "wg": normal(f, k, scale=k ** -0.5),
             "wu": normal(f, k, scale=k ** -0.5)}
        if c["train"]:
            s["dh"] = normal(t, f, scale=0.05)
        return s
    if c["op"] == "norm":
        b, t, d = c["seqs"], c["tokens"], c["dim"]
        s = {"x": normal(b, t, d, scale=1.5), "f": None, "gate": None, "wpost": None, "wpre": None}
        if c["form"] != "pre":
            s["f"] = normal(b, t, d, scale=0.7, shift=0.1)
            s["gate"] = {"none": None, "shared": normal(d, scale=0.1, shift=0.5),
                         "sequence": normal(b, d, scale=0.3, shift=0.5)}[c["gate"]]
        if c["form"] in ("post", "both"):
            s["wpost"] = normal(d, scale=0.1, shift=1.0)
        if c["form"] != "post":
            s["wpre"] = normal(d, scale=0.1, shift=1.0)
        if c["train"]:
            s["dr"] = normal(b, t, d, scale=0.05) if c["form"] != "pre" else None
            s["dn"] = normal(b, t, d, scale=0.05) if s["wpre"] is not None else None
        return s
    # one buffer of each kind, every parameter from a whole block on; the parameters are views
    sizes = _sizes(c)
    blocks = torch.tensor([-(-n // _BLOCK) for n in sizes], device="cuda")
    first = (blocks.cumsum(0) - blocks) * _BLOCK
    rows = int(blocks.sum())
    used = torch.zeros(rows * _BLOCK + 1, device="cuda")
    used[first] = 1.0
    used.index_add_(0, first + torch.tensor(sizes, device="cuda"), torch.full((len(sizes),), -1.0, device="cuda"))
    used = used.cumsum(0)[:-1].reshape(rows, _BLOCK)
    grow = torch.rand(len(sizes), generator=g, device="cuda").mul(4).sub(2).exp() * 1e-3
    grow = torch.repeat_interleave(grow, blocks)[:, None] * used
    p = normal(rows, _BLOCK, scale=0.05, dtype=torch.float32) * used
    m = normal(rows, _BLOCK, dtype=torch.float32) * grow * 0.3
    v = (normal(rows, _BLOCK, dtype=torch.float32).square() * 0.1 + 0.9) * grow.square()
    s = {"p": p.to(dt), "g": (normal(rows, _BLOCK, dtype=torch.float32) * grow).to(dt), "step": 100}
    if c["master"]:
        s["master"] = p
    if c["bits"] == 32:
        return {**s, "m": m, "v": v}
    (mc, s["ms"]), (vc, s["vs"]) = _code_m(m), _code_v(v)
    return {**s, "mc": mc.to(torch.int8), "vc": vc.to(torch.uint8), "m": torch.empty_like(m),
            "v": torch.empty_like(v)}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] == "adamw":  # the parameters, and their moments as the framework holds them
        fm, sizes = _framework(), _sizes(case)
        blocks = [-(-n // _BLOCK) for n in sizes]
        views = {k: [a.reshape(-1)[:n] for a, n in zip(s[k].split(blocks), sizes)]
                 for k in ("p", "g", "m", "v", "master", "mc", "vc") if k in s}
        s["values"] = views["m"], views["v"]
        if case["bits"] == 8:
            for k in ("m", "v"):
                scales = s[k + "s"].reshape(-1).split(blocks)
                views[k] = [fm.Moment8(c, a) for c, a in zip(views[k + "c"], scales)]
        s["grads"] = views["g"]
        s["optimiser"] = fm.AdamW(views["p"], lr=_LR, betas=_BETAS, eps=_EPS, weight_decay=_DECAY,
                                  moments=(views["m"], views["v"]), masters=views.get("master"),
                                  step=s["step"])
    return {"case": case, **s}


# ---- plain forms -----------------------------------------------------------------------

def _act(g, act):
    """act(g) and act'(g)."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 0.134145 * g * g)


def _plain_ffn(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(g, c["act"])
    out = {"h": (a * u).to(dt)}
    if c["train"]:
        dh = s["dh"].float()
        dg, du = dh * u * da, dh * a
        out |= {"dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.t() @ x).to(dt),
                "dwu": (du.t() @ x).to(dt)}
    return out


def _standard(a, kind):
    """a without its mean (layer) over its spread, and 1 / spread, row by row."""
    if kind == "layer":
        a = a - a.mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-6)
    return a * inv, inv


def _standard_back(d, hat, inv, kind):
    d = d - hat * (d * hat).mean(-1, keepdim=True)
    return (d - d.mean(-1, keepdim=True) if kind == "layer" else d) * inv


def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    kind, scale = c["kind"], 0.5
    x, f, gate, wpost, wpre = (None if s[k] is None else s[k].float()
                               for k in ("x", "f", "gate", "wpost", "wpre"))
    if gate is not None and gate.dim() == 2:
        gate = gate[:, None, :]
    gs = scale if gate is None else scale * gate
    r, out = x, {}
    if f is not None:
        z, finv = (f, None) if wpost is None else _standard(f, kind)
        fhat = z
        z = z if wpost is None else z * wpost
        r = x + gs * z
        out["r"] = r.to(dt)
    if wpre is not None:
        rhat, rinv = _standard(r, kind)
        out["n"] = (rhat * wpre).to(dt)
    if not c["train"]:
        return out
    dr = 0 if s["dr"] is None else s["dr"].float()
    if wpre is not None:
        dn = s["dn"].float()
        out["dwpre"] = (dn * rhat).sum((0, 1)).to(dt)
        dr = dr + _standard_back(dn * wpre, rhat, rinv, kind)
    out["dx"] = dr.to(dt)
    if f is not None:
        dz = gs * dr
        if gate is not None:
            out["dgate"] = (scale * z * dr).sum(1 if s["gate"].dim() == 2 else (0, 1)).to(dt)
        if wpost is not None:
            out["dwpost"] = (dz * fhat).sum((0, 1)).to(dt)
            dz = _standard_back(dz * wpost, fhat, finv, kind)
        out["df"] = dz.to(dt)
    return out


def _scale(top):
    """A block's scale (its largest magnitude; 0 below the least normal number) and its reciprocal."""
    tiny = top < torch.finfo(torch.float32).tiny
    return torch.where(tiny, 0, top), torch.where(tiny, 0, 1 / top)


def _code_m(m):
    a, inv = _scale(m.abs().amax(1, keepdim=True))
    return torch.sign(m) * torch.round(torch.sqrt(m.abs() * inv) * 127.0), a


def _code_v(v):
    a, inv = _scale(v.amax(1, keepdim=True))
    q = v * inv
    c = torch.round(torch.sqrt(torch.sqrt(q)) * 255.0)
    return torch.where(q > 0, torch.clamp(c, min=1.0), c), a


def _value_m(c, a):
    t = c * (1.0 / 127.0)
    return torch.sign(c) * (t * t) * a


def _value_v(c, a):
    t = c * (1.0 / 255.0)
    t = t * t
    return (t * t) * a


def _plain_adamw(s):
    c = s["case"]
    s["step"] += 1
    (b1, b2), t = _BETAS, s["step"]
    p, g = (s["master"] if c["master"] else s["p"]).float(), s["g"].float()
    m, v = s["m"], s["v"]
    if c["bits"] == 8:
        m, v = _value_m(s["mc"].float(), s["ms"]), _value_v(s["vc"].float(), s["vs"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    den = torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** t)) + _EPS
    p = p * (1 - _LR * _DECAY) - (m / den) * (_LR / (1 - b1 ** t))
    s["p"] = p.to(_TYPES[c["dtype"]])
    if c["master"]:
        s["master"] = p
    if c["bits"] == 8:
        (mc, s["ms"]), (vc, s["vs"]) = _code_m(m), _code_v(v)
        m, v = _value_m(mc, s["ms"]), _value_v(vc, s["vs"])
        s["mc"], s["vc"] = mc.to(torch.int8), vc.to(torch.uint8)
    s["m"], s["v"] = m, v
    return _stepped(s)


def _stepped(s):
    """What a step leaves: parameters, the moments' values, masters."""
    return {k: s[k] for k in ("p", "m", "v", "master") if k in s}


# ---- the framework's operators ---------------------------------------------------------

def _own_ffn(s):
    fm, c = _framework(), s["case"]
    out = {"h": fm.gated_ffn_forward(s["x"], s["wg"], s["wu"], c["act"])}
    if c["train"]:
        out["dx"], out["dwg"], out["dwu"] = fm.gated_ffn_pullback(s["dh"], s["x"], s["wg"], s["wu"],
                                                                  c["act"])
    return out


def _own_norm(s):
    fm, c = _framework(), s["case"]
    args = dict(gate=s["gate"], post_weight=s["wpost"], pre_weight=s["wpre"], scale=0.5,
                kind=c["kind"], eps=1e-6)
    r, n = fm.block_norm_forward(s["x"], s["f"], **args)
    out = {"r": None if s["f"] is None else r, "n": n}
    if c["train"]:
        out["dx"], out["df"], out["dgate"], out["dwpost"], out["dwpre"] = fm.block_norm_pullback(
            s["dr"], s["dn"], s["x"], s["f"], **args)
    return {k: v for k, v in out.items() if v is not None}


def _own_adamw(s):
    s["optimiser"].step(s["grads"])
    if s["case"]["bits"] == 8:
        s["optimiser"].moment_values(out=s["values"])
    return _stepped(s)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"ffn": _own_ffn, "norm": _own_norm, "adamw": _own_adamw}[op](state)
    return {"ffn": _plain_ffn, "norm": _plain_norm, "adamw": _plain_adamw}[op](state)


# ---- 64 bits ---------------------------------------------------------------------------

def exact(case, seed):
    """The definitions in 64 bits, gradients by differentiating the definition."""
    s, c = _inputs(case, seed), case
    wide = lambda t: None if t is None else t.double()  # noqa: E731
    if c["op"] == "ffn":
        x, wg, wu = (wide(s[k]).requires_grad_(c["train"]) for k in ("x", "wg", "wu"))
        g = torch.nn.functional.linear(x, wg)
        if c["act"] == "silu":
            a = g * torch.sigmoid(g)
        elif c["act"] == "gelu":
            a = g * torch.special.ndtr(g)
        else:
            a = g * torch.sigmoid(math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3))
        h = a * torch.nn.functional.linear(x, wu)
        out = {"h": h.detach()}
        if c["train"]:
            out["dx"], out["dwg"], out["dwu"] = torch.autograd.grad(h, (x, wg, wu), wide(s["dh"]))
        return out
    if c["op"] == "norm":
        names = [k for k in ("x", "f", "gate", "wpost", "wpre") if s[k] is not None]
        v = {k: wide(s[k]).requires_grad_(c["train"]) for k in names}
        d = c["dim"]

        def norm(a, w):
            centre = a.mean(-1, keepdim=True) if c["kind"] == "layer" else 0.0
            a = a - centre
            return a * (a.pow(2).sum(-1, keepdim=True) / d + 1e-6).rsqrt() * w

        out, r = {}, v["x"]
        if "f" in v:
            z = norm(v["f"], v["wpost"]) if "wpost" in v else v["f"]
            if "gate" in v:
                z = z * (v["gate"].unsqueeze(1) if v["gate"].dim() == 2 else v["gate"])
            r = r + 0.5 * z
            out["r"] = r
        if "wpre" in v:
            out["n"] = norm(r, v["wpre"])
        if c["train"]:
            outs = [out[k] for k in ("r", "n") if k in out]
            into = [wide(s["d" + k]) for k in ("r", "n") if k in out]
            grads = torch.autograd.grad(outs, list(v.values()), into)
            out |= {"d" + k: t for k, t in zip(v, grads)}
        return {k: t.detach() for k, t in out.items()}
    t, (b1, b2) = s["step"] + 1, _BETAS
    g, p = s["g"].double(), s["master" if c["master"] else "p"].double()
    m, v = s["m"].double(), s["v"].double()
    if c["bits"] == 8:
        m = s["mc"].double() * s["mc"].double().abs() / 127 ** 2 * s["ms"].double()
        v = (s["vc"].double() / 255) ** 4 * s["vs"].double()
    m, v = torch.lerp(g, m, b1), torch.lerp(g ** 2, v, b2)
    p = p - _LR * (_DECAY * p + m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + _EPS))
    out = {"p": p, "m": m, "v": v} if c["bits"] == 32 else {"p": p, "m": None, "v": None}
    if c["master"]:
        out["master"] = p
    return out
