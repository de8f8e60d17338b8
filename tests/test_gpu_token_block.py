"""The operators of a token block together: the example's training run, and its gradients
against the same block written in torch operations."""
import importlib.util
import os

import pytest
import torch

import flashmaxsim as fm

pytestmark = pytest.mark.gpu
EXAMPLE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                       "train_token_block.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_token_block", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits", [32, 8])
def test_training_lowers_the_loss(example, device, bits):
    losses, _ = example.train(40, bits, device=device, batch=32, doc_len=60, dim=128, hidden=256, embed=64)
    assert torch.isfinite(losses).all()
    assert losses[-5:].mean() < 0.7 * losses[:5].mean()


def test_block_gradients_match_torch(example, device):
    """fp32: two roundings' worth of difference at most over sums of a few hundred terms."""
    block = example.TokenBlock(48, 80, 32, torch.float32, device)
    x = torch.randn(3, 7, 48, device=device)
    up = torch.randn(3, 7, 32, device=device)
    (block(x) * up).sum().backward()
    got = [p.grad.clone() for p in block.parameters()]
    for p in block.parameters():
        p.grad = None

    def norm(a, w):
        return a / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-6) * w

    n = norm(x, block.first)
    f = (torch.nn.functional.silu(n @ block.wg.t()) * (n @ block.wu.t())) @ block.wd.t()
    e = norm(x + block.gate * norm(f, block.post), block.last) @ block.proj.t()
    (e / e.norm(dim=-1, keepdim=True) * up).sum().backward()
    for g, p in zip(got, block.parameters()):
        torch.testing.assert_close(g, p.grad, rtol=2e-4, atol=2e-4)


def test_a_query_is_encoded_as_in_its_batch(example, device):
    """Serving: a query alone (few tokens) gets the embeddings it gets among others, to one
    rounding of the feature type in the block's sums."""
    block = example.TokenBlock(256, 512, 128, torch.float16, device)
    q = torch.randn(40, 32, 256, device=device).half()
    with torch.no_grad():
        whole, alone = block(q), block(q[3:4])
    assert (whole[3:4].float() - alone.float()).abs().max() <= 4e-3


def test_second_derivatives_are_refused(device):
    """The pullbacks are not differentiable themselves, and say so."""
    x = torch.randn(4, 32, device=device, requires_grad=True)
    w = torch.randn(8, 32, device=device)
    for y in (fm.gated_ffn(x, w, w), fm.block_norm(x, pre_weight=w[0])[1]):
        (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_a_parameter_given_twice_is_refused(device):
    p = torch.zeros(8, device=device)
    with pytest.raises(fm.ArgumentError):
        fm.AdamW([p, p])
