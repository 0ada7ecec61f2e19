"""token_losses' kernels where the vocabulary goes by in pieces and dh's sums are cut as well, on FP32's tiles of 128 over many steps,
and on large tiles of rows that are no whole 16-byte pieces: against the definition in 64 bits."""

import pytest
import torch

import adambridge_amd as ab
from test_token_losses_gpu import BF16, FP32, _check, _definition, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


# 4096 rows of 70001 words are two pieces of G, which a few tiles of dh add to in nine parts (FP32 three)
@pytest.mark.parametrize("dtype,size", [(BF16, 264), (BF16, 267), (FP32, 130)])
def test_pieces_of_the_vocabulary_in_parts(dtype, size):
    gen = torch.Generator("cuda").manual_seed(size)
    _check(*_inputs(4096, 70001, size, dtype, gen))


# 66000 rows of which some 200 are scored: pieces of 4096 words, whose last one has one word, fewer than dh's parts
@pytest.mark.parametrize("dtype,size", [(BF16, 72), (BF16, 75), (FP32, 70)])
def test_a_last_piece_of_fewer_words_than_parts(dtype, size):
    rows, vocab = 66000, 61441
    gen = torch.Generator("cuda").manual_seed(size)
    h, w, t, gout = _inputs(rows, vocab, size, dtype, gen, 0.997)
    t[7], t[rows - 1] = vocab - 1, vocab - 1   # the word of the last piece
    scored = t != -100
    assert 100 < scored.sum() < 400
    want, loss_bound, dh, dh_bound, dw, dw_bound = _definition(h[scored], w, t[scored], gout[scored], -100)
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = ab.token_losses(h, w, t)
    got = torch.autograd.grad(loss, (h, w), gout)
    assert not loss[~scored].any() and not got[0][~scored].any()
    assert ((loss.detach()[scored].double() - want).abs() <= loss_bound).all()
    assert ((got[0][scored].double() - dh).abs() <= dh_bound).all()
    assert ((got[1].double() - dw).abs() <= dw_bound).all()
    again = torch.autograd.grad(ab.token_losses(h, w, t), (h, w), gout)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


# 512 tiles of 128 and more: of the logits and dW, of the logits, of dh
@pytest.mark.parametrize("rows,vocab,size", [(1100, 8200, 1030), (3000, 3000, 333), (8200, 300, 1030), (2900, 2910, 1028)])
def test_large_fp32_tiles(rows, vocab, size):
    gen = torch.Generator("cuda").manual_seed(rows + size)
    _check(*_inputs(rows, vocab, size, FP32, gen))


# more than 128 tiles of 256 x 256: sums below and above 2048 terms
@pytest.mark.parametrize("rows,vocab,size", [(2300, 4099, 1029), (2300, 4101, 2059), (2300, 4101, 1032), (300, 33001, 267)])
def test_large_tiles_of_any_rows(rows, vocab, size):
    gen = torch.Generator("cuda").manual_seed(rows + size)
    _check(*_inputs(rows, vocab, size, BF16, gen))


# tiles of the backward pass's logits that would fit twice into the CUs' places: their sums stay whole
@pytest.mark.parametrize("rows,vocab,size,dtype", [(1000, 7000, 1032, BF16), (1000, 7000, 1029, BF16), (500, 3500, 1030, FP32)])
def test_tiles_that_would_fit_twice(rows, vocab, size, dtype):
    gen = torch.Generator("cuda").manual_seed(rows + size)
    _check(*_inputs(rows, vocab, size, dtype, gen))
