"""embed and token_losses where GPU tensors take torch operations: types, sizes and transforms that the kernels do not take, beside
the kernels' own values."""

import pytest
import torch

import adambridge_amd as ab

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 40), (torch.float32, 3), (torch.float32, 40), (torch.bfloat16, 7), (torch.float64, 9)])
def test_a_target_outside_the_vocabulary_has_gradients_of_nan(dtype, size, rows):
    """By the kernels (rows of 40 FP32 values) and by torch operations (the others) alike."""
    gen = torch.Generator("cuda").manual_seed(size)
    h, w = (torch.randn(*s, generator=gen, device="cuda").to(dtype).requires_grad_() for s in ((rows, size), (10, size)))
    t = torch.randint(0, 10, (rows,), generator=gen, device="cuda")
    t[1], t[2], t[3] = 99, -100, -1
    loss = ab.token_losses(h, w, t)
    dh, dw = torch.autograd.grad(loss.sum(), (h, w))
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[1, 3]] = True
    assert torch.equal(loss.isnan(), bad) and loss[2] == 0
    assert torch.equal(dh.isnan().all(1), bad) and torch.equal(dh.isnan().any(1), bad) and not dh[2].any() and dw.isnan().all()
    if dtype == torch.float32:
        got = torch.func.grad(lambda a, b: ab.token_losses(a, b, t).sum(), argnums=(0, 1))(h.detach(), w.detach())
        assert torch.equal(got[0].isnan(), dh.isnan()) and got[1].isnan().all()
        assert torch.allclose(got[0][~bad], dh[~bad], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -3.0])
@pytest.mark.parametrize("tokens,hidden", [(9, 40), (9, 3), (256, 33), (257, 40), (700, 2), (5000, 1030)])
def test_a_scale_that_is_not_finite_reaches_its_tokens_words_only(tokens, hidden, scale, dtype):
    """Words without tokens, the padding (the most frequent word) and ids outside the vocabulary: zeros, not -0 or NaN."""
    ids = torch.full((tokens,), 13, device="cuda")
    ids[1::3], ids[2::7], ids[3] = 4, 60, -1   # 60 words; 4 has every third token
    w = torch.randn(60, hidden, device="cuda").to(dtype).requires_grad_()
    dw, = torch.autograd.grad(ab.embed(ids, w, scale, 13), w, torch.ones(tokens, hidden, device="cuda", dtype=dtype))
    want = (torch.full((hidden,), float((ids == 4).sum()), device="cuda") * scale).to(dtype)
    assert torch.equal(dw[4].nan_to_num(), want.nan_to_num())
    others = dw[torch.arange(60, device="cuda") != 4]
    assert not others.any() and not others.signbit().any()


@pytest.mark.parametrize("rows", [6, 16, 17, 300])
def test_targets_and_ignore_indexes_at_the_ends_of_64_bits(rows):
    """A target of any 64 bits is outside the vocabulary, or is not scored where it is the ignore index."""
    gen = torch.Generator("cuda").manual_seed(rows)
    h, w = torch.randn(rows, 40, generator=gen, device="cuda"), torch.randn(700, 40, generator=gen, device="cuda")
    clean = torch.randint(0, 700, (rows,), generator=gen, device="cuda")
    want = ab.token_losses(h, w, clean)
    ends = [-(1 << 63), 1 - (1 << 63), (1 << 63) - 1, -(1 << 32), 1 << 32]
    t = clean.clone()
    t[:5] = torch.tensor(ends, device="cuda")
    for ignore in (-100, *ends):
        loss = ab.token_losses(h, w, t, ignore)
        assert torch.equal(loss[5:], want[5:])
        assert [x.isnan().item() for x in loss[:5]] == [end != ignore for end in ends] and all(x == 0 or x.isnan() for x in loss[:5])
    for ignore in (1 << 40, -(1 << 40)):
        assert torch.equal(ab.token_losses(h, w, clean.int(), ignore), want)
