"""Trains a token block under MaxSim, every operator on the library's HIP kernels.

An encoder's token states (synthetic here) become embeddings through one residual block:

    n    = norm(x)                                         block_norm
    f    = (silu(n wg^T) * (n wu^T)) wd^T                  gated_ffn, then a plain product
    r, n = x + gate * norm(f), norm(r)                     block_norm
    e    = n proj^T, unit length

Queries and documents are scored with in-batch MaxSim, a softmax loss picks each query's own
document, MaxSim's pullback carries the gradients back through the block, and AdamW with 8-bit
moments over fp32 masters takes the step.

    python examples/train_token_block.py [--steps 60] [--bits 8]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "flashmaxsim.jl_amd"))
import flashmaxsim as fm  # noqa: E402


class TokenBlock:
    """Parameters of the block, 16-bit, on the device."""

    def __init__(self, dim, hidden, embed, dtype, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def matrix(rows, cols):
            return torch.randn(rows, cols, generator=g, device=device) * cols ** -0.5

        self.wg, self.wu = matrix(hidden, dim), matrix(hidden, dim)
        self.wd, self.proj = matrix(dim, hidden), matrix(embed, dim)
        self.first, self.post, self.last = (torch.ones(dim, device=device) for _ in range(3))
        self.gate = torch.full((dim,), 0.1, device=device)
        for name, p in vars(self).items():
            setattr(self, name, p.to(dtype).requires_grad_())

    def parameters(self):
        return list(vars(self).values())

    def __call__(self, x):
        """x (B, T, dim) -> unit embeddings (B, T, embed)."""
        _, n = fm.block_norm(x, pre_weight=self.first)
        h = fm.gated_ffn(n, self.wg, self.wu)
        f = (h.flatten(0, 1) @ self.wd.t()).view_as(x)
        _, n = fm.block_norm(x, f, gate=self.gate, post_weight=self.post, pre_weight=self.last)
        e = (n.flatten(0, 1) @ self.proj.t()).view(*x.shape[:2], -1).float()
        return (e / e.norm(dim=-1, keepdim=True).clamp_min(1e-6)).to(x.dtype)


def batches(batch, query_len, doc_len, dim, dtype, device, topics=16, noise=2.0, seed=1):
    """Endless (query states, document states).  A state is a point of a few topic dimensions
    under noise in all; document i holds the topics of query i, and others, under its own
    noise.  The block learns to see the topics."""
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    basis = normal(topics, dim) * topics ** -0.5
    while True:
        own, rest = normal(batch, query_len, topics), normal(batch, doc_len - query_len, topics)
        states = torch.cat([own, own, rest], 1).flatten(0, 1) @ basis
        states = states.view(batch, -1, dim) + noise * normal(batch, query_len + doc_len, dim)
        q, d = states.to(dtype).split([query_len, doc_len], 1)
        yield q.contiguous(), d.contiguous()


def train(steps, bits=8, dtype=torch.bfloat16, device="cuda:0", batch=64, query_len=32, doc_len=180,
          dim=256, hidden=512, embed=128, lr=2e-3, log=None):
    """The losses of the steps, and the block."""
    block = TokenBlock(dim, hidden, embed, dtype, device)
    optimiser = fm.AdamW(block.parameters(), lr=lr, weight_decay=1e-2, bits=bits, masters=True)
    target = torch.arange(batch, device=device)
    losses = []
    for step, (q, d) in zip(range(steps), batches(batch, query_len, doc_len, dim, dtype, device)):
        scores = fm.maxsim(block(q), block(d), fm.InBatch())  # (queries, documents)
        loss = torch.nn.functional.cross_entropy(scores, target)
        for p in block.parameters():
            p.grad = None
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
        if log and (step % 10 == 0 or step + 1 == steps):
            hit = (scores.argmax(1) == target).float().mean()
            log(f"step {step:4d}  loss {float(loss.detach()):.4f}  own document first {float(hit):.3f}")
    return torch.stack(losses), block


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--bits", type=int, default=8, choices=(8, 32), help="of AdamW's moments")
    args = parser.parse_args()
    train(args.steps, args.bits, log=lambda line: print(line, flush=True))
