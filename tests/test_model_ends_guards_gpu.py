"""embed and token_losses by their C entry points between guards: operands inside a buffer of NaN, at any element's address, results
and scratch inside one of a value that no call writes."""

import pytest
import torch

import adambridge_amd as ab
from test_operator_guards_gpu import CODES, GUARD, _call, _inside, _Result, _work
from test_token_losses_gpu import _definition

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def _untouched(work):
    assert (work.whole[:GUARD] == -7).all() and (work.whole[GUARD + work.n:] == -7).all()


# rows of less than a vector, of whole ones and not; tokens without a sort, of one run and of several
@pytest.mark.parametrize("shift", [0, 1, 5])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tokens,vocab,hidden", [
    (1, 1, 1), (5, 7, 33), (70, 3, 3), (200, 40, 9), (256, 700, 136), (257, 50, 130), (300, 5, 5), (700, 9, 2), (4097, 33, 1030), (5000, 300, 7),
    (5000, 17, 4099), (70001, 33, 12)])
def test_embed(tokens, vocab, hidden, dtype, shift):
    gen = torch.Generator("cuda").manual_seed(tokens + hidden)
    weight = torch.randn(vocab, hidden, generator=gen, device="cuda").to(dtype).requires_grad_()
    ids = (torch.randint(-1, vocab + 1, (tokens,), generator=gen, device="cuda") * torch.randint(0, 2, (tokens,), generator=gen, device="cuda"))
    g = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype)
    padding = vocab - 1
    y = ab.embed(ids, weight, 1.5, padding)
    dw, = torch.autograd.grad(y, weight, g)
    wi, gi = _inside(weight.detach(), shift), _inside(g, shift)
    for where in (ids, ids.int()):
        ii, out, grad = _inside(where, 1), _Result(y.shape, dtype, shift), _Result(dw.shape, dtype, shift)
        _call("adambridge_embed", ii, where.element_size(), tokens, wi, CODES[dtype], vocab, hidden, 1.5, out)
        out.check(y.detach(), dict(rtol=0, atol=0, equal_nan=True))
        work = _work("adambridge_embed_work", tokens, vocab, hidden)
        _call("adambridge_embed_backward", ii, where.element_size(), tokens, gi, CODES[dtype], vocab, hidden, 1.5, padding, grad, work)
        grad.check(dw)
        _untouched(work)


# rows that stream the weights; small, large and FP32 tiles; sums in parts; pieces of the vocabulary; a large part not scored
@pytest.mark.parametrize("shift", [0, 1, 5])
@pytest.mark.parametrize("rows,vocab,size,dtype", [
    (1, 1, 8, BF16), (9, 700, 40, BF16), (16, 65, 33, BF16), (16, 1001, 33, FP32), (17, 65, 264, BF16), (300, 257, 100, BF16), (300, 257, 101, FP32),
    (51, 74, 2056, BF16), (64, 37, 1030, BF16), (64, 37, 1030, FP32), (2300, 4099, 1029, BF16), (2300, 4099, 2056, BF16), (1100, 8200, 90, FP32),
    (66000, 4100, 8, BF16), (5, 9, 4, FP32)])
def test_token_losses(rows, vocab, size, dtype, shift):
    gen = torch.Generator("cuda").manual_seed(rows + vocab)
    h = torch.randn(rows, size, generator=gen, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(vocab, size, generator=gen, device="cuda") * size ** -0.5).to(dtype).requires_grad_()
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    t[::3] = -100 if rows > 1 else 0
    gout = torch.rand(rows, generator=gen, device="cuda")
    want = ab.token_losses(h, w, t)
    want_h, want_w = torch.autograd.grad(want, (h, w), gout)
    # operands at another address may take another kernel: whole 16-byte pieces or not, the same sums in another order
    if shift:
        exact, loss_bound, dh, dh_bound, dw, dw_bound = _definition(h.detach(), w.detach(), t, gout, -100)
        bounds = {id(want): (exact, loss_bound), id(want_h): (dh, dh_bound), id(want_w): (dw, dw_bound)}

    def check(result, expected):
        result.check(result.value, dict(equal_nan=True))   # the guards
        if shift:
            exact, bound = bounds[id(expected)]
            assert ((result.value.double() - exact).abs() <= bound).all()
        else:
            assert torch.equal(result.value, expected.detach())

    code, (hi, wi, gi, ti) = CODES[dtype], (_inside(x.detach(), s) for x, s in ((h, shift), (w, shift), (gout, shift), (t, 1)))
    losses, stats = _Result((rows,), FP32, shift), _Result((rows, 2), FP32, shift)
    work = _work("adambridge_token_losses_work", code, rows, vocab, size)
    _call("adambridge_token_losses", hi, wi, code, ti, rows, vocab, size, -100, losses, stats, work)
    check(losses, want)
    stats.check(stats.value, dict(equal_nan=True))
    _untouched(work)
    work = _work("adambridge_token_losses_backward_work", code, rows, vocab, size)
    for wanted in ((True, True), (True, False), (False, True)):
        outs = [_Result(x.shape, dtype, shift) if wants else None for x, wants in zip((want_h, want_w), wanted)]
        _call("adambridge_token_losses_backward", gi, hi, wi, code, ti, rows, vocab, size, -100, stats, *outs, work)
        for out, expected in zip(outs, (want_h, want_w)):
            if out is not None:
                check(out, expected)
        _untouched(work)
