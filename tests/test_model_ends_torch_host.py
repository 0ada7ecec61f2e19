"""embed, token_losses and expert_mlp in torch operations: values, gradients and refusals where they differ from the kernels' most easily."""

import pytest
import torch

import adambridge_amd as ab
from adambridge_amd.vocabulary import BACKWARD


def _same(got, want):
    """NaN at the same places, the others alike (FP32 sums of a few terms, in another order)."""
    return torch.equal(got.isnan(), want.isnan()) and torch.allclose(got.nan_to_num(), want.nan_to_num(), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
def test_a_target_outside_the_vocabulary_has_gradients_of_nan(dtype):
    gen = torch.Generator().manual_seed(0)
    h, w = (torch.randn(*s, generator=gen).to(dtype).requires_grad_() for s in ((5, 6), (10, 6)))
    t, g = torch.tensor([1, 99, -100, -1, 4]), torch.rand(5, generator=gen)
    loss = ab.token_losses(h, w, t)
    dh, dw = torch.autograd.grad(loss, (h, w), g.to(loss.dtype))
    bad = torch.tensor([False, True, False, True, False])
    assert torch.equal(loss.isnan(), bad) and loss[2] == 0
    assert torch.equal(dh.isnan().all(1), bad) and torch.equal(dh.isnan().any(1), bad) and not dh[2].any() and dw.isnan().all()
    alone = torch.autograd.grad(ab.token_losses(h, w, torch.where(bad, -100, t)), h, g.to(loss.dtype))[0]
    assert torch.equal(dh[~bad], alone[~bad])
    if dtype == torch.float32:
        want = BACKWARD["token_losses"](g, h.detach(), w.detach(), t, -100, True, True)
        assert _same(dh, want[0]) and _same(dw, want[1])
        got = torch.func.grad(lambda a, b: (ab.token_losses(a, b, t) * g).sum(), argnums=(0, 1))(h.detach(), w.detach())
        assert _same(got[0], dh) and _same(got[1], dw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_a_logit_of_inf_leaves_no_distribution(dtype):
    """Losses and gradients of NaN, whether or not it is the target's; a word that no row can reach (-inf) leaves the others' losses."""
    h, w = torch.ones(4, 6, dtype=dtype), torch.randn(10, 6, generator=torch.Generator().manual_seed(1)).to(dtype)
    t = torch.tensor([1, 3, 2, -100])
    w[3, 0] = torch.inf
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = ab.token_losses(h, w, t)
    assert torch.equal(loss.isnan(), t != -100)
    assert torch.equal(torch.autograd.grad(loss.sum(), h)[0].isnan().any(1), t != -100)
    with torch.no_grad():
        w[3, 0] = -torch.inf
    loss = ab.token_losses(h, w, t)
    want = ab.token_losses(h[0], torch.cat((w[:3], w[4:])), torch.tensor(1))
    assert torch.allclose(loss[0], want) and loss[1] == torch.inf and loss[3] == 0
    assert ab.token_losses(h, torch.full_like(w, -torch.inf), t)[:3].isnan().all()


def test_a_row_that_is_not_scored_reaches_nothing_beside_an_infinite_weight():
    """A word of inf that the scored rows hold at -inf: their losses are finite, and so are the weight's gradients; a row that is not
    scored has a gradient of zeros."""
    h, w = -torch.ones(4, 6), torch.randn(10, 6, generator=torch.Generator().manual_seed(2))
    h[3] = torch.nan
    w[3, 0] = torch.inf
    t, g = torch.tensor([1, 2, -100, -100]), torch.rand(4, generator=torch.Generator().manual_seed(3))
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = ab.token_losses(h, w, t)
    assert loss[:2].isfinite().all() and not loss[2:].any()
    for dh, dw in (torch.autograd.grad(loss, (h, w), g), BACKWARD["token_losses"](g, h.detach(), w.detach(), t, -100, True, True)[:2]):
        assert not dh[2:].any() and dw.isfinite().all() and not dw[3].any()
    loss = ab.token_losses(h, w, torch.full_like(t, -100))
    assert not loss.any() and all(not x.any() for x in torch.autograd.grad(loss.sum(), (h, w)))


def test_an_ignore_index_that_is_no_target_s_type():
    """One past 32 bits ignores no row of int32 targets; one past 64 bits is refused."""
    gen = torch.Generator().manual_seed(4)
    h, w, t = torch.randn(4, 6, generator=gen), torch.randn(10, 6, generator=gen), torch.tensor([0, 1, 2, 3])
    want = ab.token_losses(h, w, t)
    for ignore in (1 << 32, 1 << 40, -(1 << 40), (1 << 63) - 1, -(1 << 63)):
        assert torch.equal(ab.token_losses(h, w, t.int(), ignore), want) and torch.equal(ab.token_losses(h, w, t, ignore), want)
    assert (want > 0).all()
    for ignore in (1 << 63, -(1 << 63) - 1, 1 << 70):
        for targets in (t, t.int()):
            with pytest.raises(ValueError, match="ignore_index must be an int of 64 bits"):
                ab.token_losses(h, w, targets, ignore)


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -3.0])
def test_a_scale_that_is_not_finite_reaches_its_tokens_words_only(scale):
    """Words without tokens, the padding and ids outside the vocabulary: zeros."""
    w, ids = torch.randn(5, 4, requires_grad=True), torch.tensor([1, -1, 7, 2, 1])
    y = ab.embed(ids, w, scale, 2)
    assert torch.equal(y[[0, 3, 4]].detach().nan_to_num(), (w.detach()[[1, 2, 1]] * scale).nan_to_num())
    for dw in (torch.autograd.grad(y, w, torch.ones(5, 4))[0], BACKWARD["embed"](torch.ones(5, 4), ids, 5, scale, 2)[1]):
        assert not dw[[0, 2, 3, 4]].any() and torch.equal(dw[1].nan_to_num(), torch.full((4,), 2 * scale).nan_to_num())


def test_a_vocabulary_past_32_bits_with_int32_ids():
    """(One row of memory.)"""
    weight = torch.full((1, 2), 3.0).expand((1 << 32) + 9, 2)
    ids = torch.tensor([0, 7, 8, 9, (1 << 31) - 1, -1], dtype=torch.int32)
    assert torch.equal(ab.embed(ids, weight).isnan().all(1), ids < 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_few_tokens_without_gradients_do_not_widen_the_table(dtype, monkeypatch):
    """With a gradient the whole table is taken in FP32, in which its rows' gradients are summed."""
    weight, ids = torch.randn(500, 8).to(dtype).requires_grad_(), torch.tensor([3, 499, 500, 3])
    sizes, to = [], torch.Tensor.to
    monkeypatch.setattr(torch.Tensor, "to", lambda self, *args, **kwargs: (sizes.append(self.numel()), to(self, *args, **kwargs))[1])
    trained = ab.embed(ids, weight, 1.7, 3)
    assert max(sizes) == 4000
    sizes.clear()
    with torch.no_grad():
        rows = ab.embed(ids, weight, 1.7, 3)
    assert torch.equal(ab.embed(ids, weight.detach(), 1.7, 3).nan_to_num(), rows.nan_to_num()) and max(sizes) <= 32
    assert torch.equal(rows.nan_to_num(), trained.detach().nan_to_num())
