"""embed, token_losses and expert_mlp at the ends of the sizes that they take, each alone: rows, words, values of a row."""

import pytest
import torch

import adambridge_amd as ab
from test_expert_mlp_gpu import BF16, FP32, _check as _check_mlp
from test_token_losses_gpu import _check as _check_losses, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


# the most rows, words (streamed, on tiles) and values of a row (whole 16-byte pieces and not)
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,vocab,size", [(1 << 23, 3, 8), (4, 1 << 22, 8), (20, (1 << 22) - 3, 9), (3, 70, 1 << 20), (2, 5, (1 << 20) - 1)])
def test_token_losses(rows, vocab, size, dtype):
    gen = torch.Generator("cuda").manual_seed(rows + size)
    h, w, t, gout = _inputs(rows, vocab, size, dtype, gen)
    t[0] = vocab - 1
    _check_losses(h, w, t, gout)


@pytest.mark.parametrize("size", ["rows", "words", "values"])
def test_token_losses_past_the_largest_take_torch_operations(size):
    """One more of each than the kernels take (the weight of one row of memory)."""
    if size == "rows":
        h, w, t = torch.zeros((1 << 23) + 1, 4, device="cuda"), torch.randn(2, 4, device="cuda"), torch.zeros((1 << 23) + 1, dtype=torch.int64, device="cuda")
    elif size == "words":
        h, w, t = torch.zeros(2, 4, device="cuda"), torch.randn(1, 4, device="cuda").expand((1 << 22) + 1, 4), torch.tensor([0, 1 << 22], device="cuda")
    else:
        h, w, t = torch.zeros(2, (1 << 20) + 1, device="cuda"), torch.randn(3, (1 << 20) + 1, device="cuda"), torch.tensor([0, 2], device="cuda")
    want = torch.full(t.shape, float(w.shape[0]), device="cuda").log()
    assert torch.allclose(ab.token_losses(h, w, t), want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tokens", [5, 300])
@pytest.mark.parametrize("hidden", [1 << 22, (1 << 22) - 1])
def test_embed(hidden, tokens, dtype):
    """Gradients of whole numbers, whose sums FP32 holds; of 300 tokens most are one word's."""
    gen = torch.Generator("cuda").manual_seed(tokens)
    ids = torch.zeros(tokens, dtype=torch.int64, device="cuda")
    ids[1::9], ids[2] = 2, 3
    weight = torch.randn(3, hidden, generator=gen, device="cuda").to(dtype).requires_grad_()
    y = ab.embed(ids, weight, 2.0)
    assert torch.equal(y[:2], weight[ids[:2]] * 2.0) and y[2].isnan().all() and torch.equal(y[-1], weight[ids[-1]] * 2.0)
    del y
    g = torch.randint(-3, 4, (tokens, hidden), generator=gen, device="cuda", dtype=torch.int8).to(dtype)
    dw, = torch.autograd.grad(ab.embed(ids, weight, 2.0), weight, g)
    for word in range(3):
        assert torch.equal(dw[word], (g[ids == word].float().sum(0) * 2.0).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("experts,inter,hidden", [(1, 1, 1 << 22), (2, 9, (1 << 22) - 1), (2, 1 << 22, 8), (1, (1 << 22) - 1, 3)])
def test_expert_mlp(experts, inter, hidden, dtype):
    gen = torch.Generator("cuda").manual_seed(experts + inter)
    _check_mlp(3, experts, 1, inter, hidden, dtype, True, "silu", True, gen)
    _check_mlp(16, experts, experts, inter, hidden, dtype, False, "gelu", False, gen)
