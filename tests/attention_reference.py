"""Attention over heads in 64 bits, written from its definition, and how far results rounded once may be
from it: every entry comes with a bound of what fp32 sums and the roundings to the feature type cost."""
import torch


def counts(nq, nk, causal=False, window=None, device="cpu"):
    """(nq, nk): which keys a query sees by position, the last ones beside one another."""
    away = torch.arange(nk, device=device)[None] - torch.arange(nq, device=device)[:, None] - (nk - nq)
    keep = torch.ones(nq, nk, dtype=torch.bool, device=device)
    if causal:
        keep &= away <= 0
    if window is not None:
        keep &= away.abs() <= window
    return keep


def reference(q, k, v, keep, scale, do=None):
    """One sequence: q (Tq, H, d), k and v (Tk, Hk, d), keep (Tq, Tk).  Returns {name: (value, bound)} for
    o and, with do, dq, dk and dv."""
    if 0 in (*q.shape, *k.shape):  # sums of nothing
        none = {"o": q, "dq": q, "dk": k, "dv": k}
        return {name: (torch.zeros_like(t, dtype=torch.float64), torch.ones_like(t, dtype=torch.float64) * 1e-300)
                for name, t in none.items()}
    half = torch.finfo(q.dtype).eps / 2
    # (half a step among the feature type's smallest numbers)
    floor = torch.finfo(q.dtype).smallest_normal * half
    H, Hk, d = q.shape[1], k.shape[1], q.shape[2]
    group = H // Hk
    nq, nk = q.shape[0], k.shape[0]
    # masked places may hold anything
    qs, ks = keep.any(1), keep.any(0)
    wide = lambda t, ok: torch.where(ok[:, None, None], t.double(), 0.0).transpose(0, 1)  # noqa: E731
    Q, K, V = wide(q, qs), wide(k, ks).repeat_interleave(group, 0), wide(v, ks).repeat_interleave(group, 0)
    s = (Q @ K.transpose(1, 2).contiguous()) * scale
    s = s.masked_fill(~keep, -float("inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    # What a p may be off by, relative to itself, before it is rounded: the score's sum of d products, its
    # product with scale * log2 e, the maximum's or the logarithm's own rounding, the exponential (2 units).
    unit = 2.0 ** -24
    size = (abs(scale) * (Q.abs() @ K.abs().transpose(1, 2).contiguous())).masked_fill(~keep, 0.0)
    rows = size.amax(-1, keepdim=True)
    off = unit * ((d + 4) * rows + 16) * 2 + unit * (nk + 64)
    # p in its product: in 16 bits a rounding and what it left, itself rounded; small fp16 ones on a grid of 2^-24,
    # scaled by 2^10 or more
    rough = half * half if q.dtype != torch.float32 else 0.0
    grid = 2.0 ** -35 if q.dtype == torch.float16 else 0.0
    o = p @ V
    mass = p @ V.abs()
    out = {"o": (o, half * o.abs() + (rough * 1.01 + off) * mass + grid * V.abs().sum(1, keepdim=True) + floor)}
    if do is not None:
        D = wide(do, qs)
        dv = p.transpose(1, 2).contiguous() @ D
        dp = D @ V.transpose(1, 2).contiguous()
        delta = (p * dp).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # dp and delta are fp32 sums; delta's o has what its rounding left, to the square of the rounding, and the
        # error of its p
        dp_size = D.abs() @ V.abs().transpose(1, 2).contiguous()
        delta_size = (p * dp_size).sum(-1, keepdim=True)
        delta_off = ((unit * (d + nk + 64) + 4 * half * half) * delta_size + off * delta_size
                     + rough * 1.01 * delta_size
                     + grid * dp_size.sum(-1, keepdim=True))
        if q.dtype == torch.float32:
            delta_off = delta_off + half * delta_size  # (o is rounded to fp32 there)
        ds_off = p * (unit * (d + 8) * (dp_size + delta_size) + delta_off) + (off + rough * 1.01) * ds.abs()
        if q.dtype == torch.float16:  # ds on its grid: 2^15 p times a factor that brings 2 |do| |v| to 1/2 at least
            bound = 2 * D.norm(dim=-1).amax(-1)[:, None, None] * V.norm(dim=-1).amax(-1)[:, None, None]
            ds_off = ds_off + 2 * bound * 2.0 ** -40
        dq, dk = scale * (ds @ K), scale * (ds.transpose(1, 2).contiguous() @ Q)
        sums = unit * (nq * group + nk + 64)
        dv_size = p.transpose(1, 2).contiguous() @ D.abs()
        dv_off = (off.amax(1, keepdim=True) + rough * 1.01 + sums) * dv_size + grid * D.abs().sum(1, keepdim=True)
        dq_off = abs(scale) * ((ds_off + sums * ds.abs()) @ K.abs())
        dk_off = abs(scale) * ((ds_off + sums * ds.abs()).transpose(1, 2).contiguous() @ Q.abs())
        share = lambda t: t.view(Hk, group, *t.shape[1:]).sum(1)  # noqa: E731
        for name, x, far in (("dq", dq, dq_off), ("dk", share(dk), share(dk_off)), ("dv", share(dv), share(dv_off))):
            out[name] = (x, half * x.abs() + 1.01 * far + floor)
    return {name: (x.transpose(0, 1), far.transpose(0, 1)) for name, (x, far) in out.items()}


def check(got, want, what):
    """Every entry within its bound."""
    x, far = want
    assert got.shape == x.shape, (what, got.shape, x.shape)
    if not got.numel():
        return
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} entries are not finite"
    over = ((got.double() - x).abs() / far).max()
    assert float(over) <= 1.0, f"{what}: {float(over):.3f} times as far off as roundings may be"
