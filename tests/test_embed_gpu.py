"""embed's kernels against 64-bit sums: sizes about the sort's runs and chunks, words of every count, ids outside the vocabulary."""

import pytest
import torch

import adambridge_amd as ab

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _ids(kind, tokens, vocab, gen):
    if kind == "same":
        return torch.full((tokens,), vocab // 2, device="cuda")
    if kind == "runs":   # long words that begin and end anywhere, and single tokens between them
        ids = (torch.arange(tokens, device="cuda") * 7919 // max(1, tokens // 5)) % vocab
        return ids[torch.randperm(tokens, generator=gen, device="cuda")]
    if kind == "outside":
        return torch.randint(-3, vocab + 3, (tokens,), generator=gen, device="cuda")
    return (torch.pow(float(vocab), torch.rand(tokens, generator=gen, device="cuda", dtype=torch.float64)) - 1).long().clamp(0, vocab - 1)


def _check(ids, vocab, hidden, dtype, scale, padding, gen):
    weight = torch.randn(vocab, hidden, generator=gen, device="cuda").to(dtype).requires_grad_()
    y = ab.embed(ids, weight, scale, padding)
    inside = (ids >= 0) & (ids < vocab)
    at = torch.where(inside, ids, 0).long()
    want = torch.where(inside[..., None], weight.detach()[at].float() * torch.tensor(scale, device="cuda"), torch.nan).to(dtype)
    assert y.dtype == dtype and y.shape == (*ids.shape, hidden)
    assert torch.equal(y.detach().nan_to_num(nan=7e4), want.nan_to_num(nan=7e4))
    g = torch.randn(y.shape, generator=gen, device="cuda").to(dtype)
    dw, = torch.autograd.grad(y, weight, g)
    counted = inside if padding is None else inside & (ids != padding)
    # on the host: adding doubles to one row from many lanes of a GPU takes minutes
    terms = torch.where(counted[..., None], g.double(), 0.0).reshape(-1, hidden).cpu()
    flat = at.reshape(-1).cpu()
    total, size = (torch.zeros(vocab, hidden, dtype=torch.float64).index_add_(0, flat, t).cuda() for t in (terms, terms.abs()))
    count = torch.bincount(flat[counted.reshape(-1).cpu()], minlength=vocab)[:, None].cuda()
    # a sum of n terms in FP32, in any order: n - 1 roundings of at most the terms' sizes; the scale's, its product's, the result's
    bound = abs(scale) * size * (count + 1) * 2.0 ** -24 + (total * scale).abs() * (2 * 2.0 ** -24 + torch.finfo(dtype).eps / 2)
    assert ((dw.double() - total * scale).abs() <= bound).all()
    assert dw.dtype == dtype and not dw[(count == 0)[:, 0]].any()
    again, = torch.autograd.grad(ab.embed(ids, weight, scale, padding), weight, g)
    assert torch.equal(again, dw)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("kind", ["words", "same", "runs", "outside"])
@pytest.mark.parametrize("tokens,vocab,hidden", [
    (1, 1, 1), (1, 50, 8), (2, 3, 9), (63, 5, 64), (64, 7, 130), (65, 7, 33), (129, 2, 513), (1000, 16, 515), (2047, 1000, 24),
    (2048, 17, 100), (2049, 300, 1030), (5000, 15, 4099), (4097, 4100, 7)])
def test_rows_and_gradients(tokens, vocab, hidden, kind, dtype):
    gen = torch.Generator("cuda").manual_seed(tokens + vocab + hidden)
    ids = _ids(kind, tokens, vocab, gen)
    _check(ids, vocab, hidden, dtype, 1.0, None, gen)
    _check(ids.int(), vocab, hidden, dtype, 1.7, vocab // 2, gen)


@pytest.mark.parametrize("kind", ["words", "same", "runs"])
@pytest.mark.parametrize("tokens,vocab,hidden", [(65536, 200, 40), (65537, 1000, 24), (70001, 33, 12), (2300003, 5000, 2)])
def test_long_batches(tokens, vocab, hidden, kind):
    """More tokens than one, and than two, merges of 32 runs take; chunks of more tokens than 64."""
    gen = torch.Generator("cuda").manual_seed(tokens)
    _check(_ids(kind, tokens, vocab, gen), vocab, hidden, FP32, -0.5, 0, gen)


def test_ids_of_any_shape_and_order():
    gen = torch.Generator("cuda").manual_seed(0)
    for ids in (torch.tensor(4, device="cuda"), torch.randint(0, 9, (3, 1, 5), device="cuda"), torch.randint(0, 9, (6, 7), device="cuda").t(),
                torch.randint(0, 9, (20,), device="cuda")[::3], torch.randint(0, 9, (5, 1), device="cuda").expand(5, 4)):
        _check(ids, 9, 20, BF16, 2.0, None, gen)
    wide = torch.randn(9, 40, device="cuda").requires_grad_()
    for weight in (wide[:, ::2], wide.t()[:20, :9].t()):
        ids, g = torch.tensor([1, 8, 1], device="cuda"), torch.randn(3, 20, device="cuda")
        y = ab.embed(ids, weight)
        assert torch.equal(y, weight[ids])
        got, want = (torch.autograd.grad(t, wide, g)[0] for t in (y, weight[ids]))
        assert torch.allclose(got, want, rtol=1e-6, atol=0)


def test_no_tokens():
    weight = torch.randn(9, 20, device="cuda", requires_grad=True)
    for shape in ((0,), (3, 0)):
        y = ab.embed(torch.empty(shape, dtype=torch.int64, device="cuda"), weight)
        assert y.shape == (*shape, 20)
        assert not torch.autograd.grad(y.sum(), weight)[0].any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("kind", ["words", "same", "outside"])
@pytest.mark.parametrize("tokens,vocab,hidden", [(255, 3, 136), (256, 700, 136), (257, 700, 136), (256, 1, 2), (200, 40000, 9)])
def test_about_the_fewest_tokens(tokens, vocab, hidden, kind, dtype):
    """Tokens that are not sorted, and the first that are."""
    gen = torch.Generator("cuda").manual_seed(tokens + vocab)
    ids = _ids(kind, tokens, vocab, gen)
    _check(ids, vocab, hidden, dtype, 1.0, None, gen)
    _check(ids.int(), vocab, hidden, dtype, 1.7, vocab - 1, gen)
