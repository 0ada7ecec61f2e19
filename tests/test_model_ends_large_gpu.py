"""Calls of embed, token_losses and expert_mlp whose arrays pass 2^31 values, or whose launches pass one dimension of a grid."""

import pytest
import torch
import torch.nn.functional as F

import adambridge_amd as ab

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def test_an_embedding_of_more_than_2_31_values():
    vocab, hidden = 540001, 4099
    weight = torch.zeros(vocab, hidden, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([0, vocab - 1, 524000, vocab - 1, 7, vocab], device="cuda")
    for i in ids[:5].tolist():
        weight[i] = torch.randn(hidden, device="cuda")
    weight.requires_grad_()
    y = ab.embed(ids, weight)
    assert torch.equal(y[:5], weight[ids[:5]]) and y[5].isnan().all()
    g = torch.randn(6, hidden, device="cuda").bfloat16()
    dw, = torch.autograd.grad(y, weight, g)
    want = {0: g[0], vocab - 1: (g[1].float() + g[3].float()).bfloat16(), 524000: g[2], 7: g[4]}
    for i, row in want.items():
        assert torch.equal(dw[i], row)
        dw[i] = 0
    assert not dw.any()


def test_tokens_of_more_than_2_31_values_and_of_more_workgroups_than_a_grid_holds():
    """Gradients of ones count the words' tokens: whole numbers, exact in FP32."""
    for tokens, vocab, hidden, dtype in ((530000, 211, 4099, torch.bfloat16), ((1 << 26) + 77, 1000, 8, torch.float32)):
        ids = torch.randint(0, vocab, (tokens,), device="cuda", dtype=torch.int32)
        weight = torch.randn(vocab, hidden, device="cuda").to(dtype).requires_grad_()
        y = ab.embed(ids, weight)
        half = tokens // 2
        for part in (slice(0, 999), slice(half, half + 999), slice(tokens - 999, tokens)):
            assert torch.equal(y[part].detach(), weight.detach()[ids[part].long()])
        g = torch.ones_like(y)
        del y
        dw, = torch.autograd.grad(ab.embed(ids, weight), weight, g)
        count = torch.bincount(ids, minlength=vocab)
        assert torch.equal(dw, count[:, None].to(dtype).expand_as(dw))


@pytest.mark.parametrize("rows,vocab", [((1 << 21) + 5, 40), (530000, 4096)])
def test_losses_of_many_rows(rows, vocab):
    """More rows than a grid holds; a piece's gradient of more than 2^31 values."""
    gen = torch.Generator("cuda").manual_seed(rows)
    h = torch.randn(rows, 8, generator=gen, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(vocab, 8, generator=gen, device="cuda").bfloat16().requires_grad_()
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    t[::3] = -100
    g = torch.rand(rows, generator=gen, device="cuda") / rows
    loss = ab.token_losses(h, w, t)
    dh, dw = torch.autograd.grad(loss, (h, w), g)
    want_dw = 0.0
    for lo in range(0, rows, 1 << 17):
        here = h.detach()[lo:lo + (1 << 17)].double().requires_grad_()
        there = w.detach().double().requires_grad_()
        want = F.cross_entropy(here @ there.t(), t[lo:lo + (1 << 17)], reduction="none")
        a, b = torch.autograd.grad(want, (here, there), g[lo:lo + (1 << 17)].double())
        # 8 products a logit, of sizes below 4 x 4; FP32's own logarithm and sums of up to 4096 exponentials
        assert torch.allclose(loss[lo:lo + (1 << 17)].detach().double(), want, rtol=2.0 ** -18, atol=2.0 ** -14)
        # the gradient at the logits is rounded to BF16, half a step of 2^-8 of each of its terms; a row's sum again
        size = 2.0 ** -7 * (g[lo:lo + (1 << 17)].double()[:, None] * 2 * w.detach().double().abs().amax(0))
        assert ((dh[lo:lo + (1 << 17)].double() - a).abs() <= size).all()
        want_dw = want_dw + b
    assert ((dw.double() - want_dw).abs() <= 2.0 ** -7 * (want_dw.abs() + 2.0 * h.detach().double().abs().mul(g.double()[:, None]).sum(0) / vocab + 1e-6)).all()


def test_experts_of_more_than_2_31_values():
    """The last expert's weights lie behind 2^31 values of both arrays."""
    experts, inter, hidden = 34, 8192, 8200
    up = torch.zeros(experts, inter, hidden, dtype=torch.bfloat16, device="cuda")
    down = torch.zeros(experts, hidden, inter, dtype=torch.bfloat16, device="cuda")
    for e in (0, experts - 1):
        up[e].normal_(0.0, 0.01)
        down[e].normal_(0.0, 0.01)
    x = torch.randn(3, hidden, device="cuda").bfloat16()
    logits = torch.full((3, experts), -9.0, device="cuda")
    logits[:, 0], logits[:, -1] = 0.5, 1.0
    out = ab.expert_mlp(x, logits, up, down, 2)
    r = ab.route(logits, 2)
    want = ab.combine(ab.expert_mm(F.gelu(ab.expert_mm(ab.dispatch(x, r), up, r.ends)), down, r.ends), r)
    assert out.float().std() > 0 and torch.allclose(out, want, rtol=2.0 ** -5, atol=2.0 ** -5 * out.float().std().item())
