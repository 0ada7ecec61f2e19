"""The example that trains and decodes with the expert block's operators together (examples/train_experts.py)."""

import importlib.util
from pathlib import Path

import pytest
import torch

import adambridge_amd as ab

_SPEC = importlib.util.spec_from_file_location("train_experts", Path(__file__).resolve().parents[1] / "examples" / "train_experts.py")
example = importlib.util.module_from_spec(_SPEC)
_SPEC.loader.exec_module(example)


def _runs(device):
    losses, model, ids = example.train(60, device, "bf16")
    assert losses[0] > 5.0 and losses[-1] < 1.0, losses   # the logarithm of 512 tokens is 6.2; the sequence repeats
    assert torch.equal(example.decode(model, ids[:24], 8), ids[24:32])


def test_the_example_learns_on_the_cpu():
    _runs("cpu")


@pytest.mark.gpu
def test_the_example_learns_on_the_gpu():
    _runs("cuda")


@pytest.mark.gpu
def test_a_block_s_gradients_on_the_gpu_are_the_cpu_s():
    """In FP32, every gradient of one block against torch operations on the CPU."""
    torch.manual_seed(1)
    block = example.ExpertBlock(64, 96, 6, 2)
    x, g = torch.randn(50, 64), torch.randn(50, 64)
    grads = []
    for device in ("cpu", "cuda"):
        here = block.to(device)
        leaf = x.to(device).requires_grad_()
        grads.append([t.cpu() for t in torch.autograd.grad(here(leaf), [leaf, *here.parameters()], g.to(device))])
    for a, b in zip(*grads):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-3 * a.abs().max().item())


@pytest.mark.gpu
def test_under_compile_and_batched_gradients():
    """A compiled block (its routing outside the graph) gives the same values; a batch of gradients takes torch
    operations, one by one the kernels'."""
    torch.manual_seed(2)
    w = torch.randn(4, 24, 32, device="cuda", requires_grad=True)
    x = torch.randn(20, 32, device="cuda", requires_grad=True)
    norm = torch.nn.LayerNorm(32).cuda()
    r = ab.route(torch.randn(20, 4, device="cuda"), 2)

    def block(t):
        return ab.combine(ab.expert_mm(ab.dispatch(ab.layer_norm(t, norm.weight, norm.bias), r), w, r.ends), r)

    want = block(x)
    got = torch.compile(block, backend="eager")(x)
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)
    g = torch.randn(3, *want.shape, device="cuda")
    one = [torch.autograd.grad(want, (x, w), v, retain_graph=True) for v in g]
    for i in range(2):
        alone, = torch.autograd.grad(want, [(x, w)[i]], g[0], retain_graph=True)
        assert torch.equal(alone, one[0][i])
    all_at_once = torch.autograd.grad(want, (x, w), g, retain_graph=True, is_grads_batched=True)
    for i in range(2):
        assert torch.allclose(all_at_once[i], torch.stack([o[i] for o in one]), rtol=1e-3, atol=1e-3)
