"""A language model's ends on the CPU: torch operations of the same values, what the calls and the C entry points refuse."""

import ctypes

import pytest
import torch

import adambridge_amd as ab
from adambridge_amd import _hip
from adambridge_amd.vocabulary import BACKWARD

EBADN, ENULL, EDTYPE, EALIGN = -1, -2, -4, -14
P = ctypes.c_void_p(256)


def test_embed_is_torch_s():
    gen = torch.Generator().manual_seed(0)
    weight = torch.randn(11, 6, generator=gen, requires_grad=True)
    ids = torch.randint(0, 11, (4, 5), generator=gen)
    g = torch.randn(4, 5, 6, generator=gen)
    y, want = ab.embed(ids, weight, 3.0, 2), torch.nn.functional.embedding(ids, weight, 2) * 3.0
    assert torch.allclose(y, want, rtol=1e-6, atol=0)
    got, expected = (torch.autograd.grad(t, weight, g)[0] for t in (y, want))
    assert torch.allclose(got, expected, rtol=1e-6, atol=1e-6) and not got[2].any()
    assert ab.embed(ids.int(), weight.bfloat16()).dtype == torch.bfloat16
    assert ab.embed(ids[:0], weight).shape == (0, 5, 6)


def test_embed_gradients():
    weight = torch.randn(7, 3, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([6, 0, 6, 3])
    assert torch.autograd.gradcheck(lambda w: ab.embed(ids, w, 1.5), (weight,))
    assert torch.autograd.gradgradcheck(lambda w: ab.embed(ids, w, 1.5), (weight,))
    got = torch.func.vmap(lambda i: ab.embed(i, weight))(torch.stack((ids, ids.flip(0))))
    assert torch.equal(got[1], weight[ids.flip(0)])


def test_embed_ids_outside_the_vocabulary():
    weight = torch.randn(5, 4, requires_grad=True)
    y = ab.embed(torch.tensor([0, -1, 5, 1 << 40, 4]), weight)
    assert y[1:4].isnan().all() and torch.equal(y[[0, 4]], weight[[0, 4]])
    dw, = torch.autograd.grad(y, weight, torch.ones(5, 4))
    assert torch.equal(dw.sum(1), torch.tensor([4.0, 0.0, 0.0, 0.0, 4.0]))


def test_embed_sums_in_32_bits():
    """4096 ones of BF16 are 4096 (in BF16 they would stay at 256)."""
    weight = torch.zeros(2, 3, dtype=torch.bfloat16, requires_grad=True)
    y = ab.embed(torch.zeros(4096, dtype=torch.int64), weight)
    assert torch.equal(torch.autograd.grad(y, weight, torch.ones_like(y))[0][0], torch.full((3,), 4096.0).bfloat16())


def test_embed_refusals():
    weight, ids = torch.randn(5, 4), torch.tensor([1, 2])
    for call, words in (
            (lambda: ab.embed(ids, weight[0]), r"\[vocab, hidden\]"),
            (lambda: ab.embed(ids, weight.long()), r"\[vocab, hidden\]"),
            (lambda: ab.embed(ids, weight[:0]), "not empty"),
            (lambda: ab.embed(ids, weight[:, :0]), "not empty"),
            (lambda: ab.embed(ids.float(), weight), "int64 or int32"),
            (lambda: ab.embed(ids.short(), weight), "int64 or int32"),
            (lambda: ab.embed(ids, weight, True), "scale must be a number"),
            (lambda: ab.embed(ids, weight, "2"), "scale must be a number"),
            (lambda: ab.embed(ids, weight, 1.0, 5), "padding_idx must be None or an int from 0 to 4"),
            (lambda: ab.embed(ids, weight, 1.0, -1), "padding_idx"),
            (lambda: ab.embed(ids, weight, 1.0, True), "padding_idx")):
        with pytest.raises(ValueError, match=words):
            call()


def test_embed_entry_points():
    """Nothing is launched for a refused call."""
    lib = _hip.open_library()
    f32 = _hip.DT_F32
    for tokens, vocab, hidden in ((0, 4, 4), ((1 << 30) + 1, 4, 4), (4, 0, 4), (4, (1 << 30) + 1, 4), (4, 4, 0), (4, 4, (1 << 22) + 1)):
        assert lib.adambridge_embed(P, 8, tokens, P, f32, vocab, hidden, 1.0, P) == EBADN
        assert lib.adambridge_embed_work(tokens, vocab, hidden) == EBADN
        assert lib.adambridge_embed_backward(P, 8, tokens, P, f32, vocab, hidden, 1.0, -1, P, P) == EBADN
    for id_bytes, dtype in ((2, f32), (8, _hip.DT_FP8), (0, f32)):
        assert lib.adambridge_embed(P, id_bytes, 4, P, dtype, 4, 4, 1.0, P) == EDTYPE
        assert lib.adambridge_embed_backward(P, id_bytes, 4, P, dtype, 4, 4, 1.0, -1, P, P) == EDTYPE
    for i in (0, 3, 8):
        args = [P, 8, 4, P, f32, 4, 4, 1.0, P]
        args[i] = None
        assert lib.adambridge_embed(*args) == ENULL
    for i in (0, 3, 9, 10):
        args = [P, 8, 4, P, f32, 4, 4, 1.0, -1, P, P]
        args[i] = None
        assert lib.adambridge_embed_backward(*args) == ENULL
    assert lib.adambridge_embed_backward(P, 8, 4, P, f32, 4, 4, 1.0, -1, P, ctypes.c_void_p(260)) == EALIGN
    # the sorted tokens twice, two parts for each of at most 2048 chunks, a place a word
    assert 0 < lib.adambridge_embed_work(1 << 20, 1000, 64) <= (1 << 20) * 16 + 2048 * 2 * 64 * 4 + 1001 * 4


# ---------------------------------------------------------------- token_losses

def test_token_losses_are_torch_s():
    gen = torch.Generator().manual_seed(1)
    h, w = torch.randn(3, 5, 6, generator=gen, requires_grad=True), torch.randn(11, 6, generator=gen, requires_grad=True)
    t = torch.randint(0, 11, (3, 5), generator=gen)
    t[1, 2:] = -100
    got = ab.token_losses(h, w, t)
    want = torch.nn.functional.cross_entropy((h @ w.t()).reshape(-1, 11), t.reshape(-1), reduction="none").view(3, 5)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-6)
    g = torch.rand(3, 5, generator=gen)
    for a, b in zip(torch.autograd.grad(got, (h, w), g), torch.autograd.grad(want, (h, w), g)):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    assert ab.token_losses(h.bfloat16(), w.bfloat16(), t.int()).dtype == torch.float32
    assert torch.equal(ab.token_losses(h, w, torch.where(t == -100, 3, t), 3) == 0, (t == -100) | (t == 3))


def test_token_losses_gradients():
    h, w = torch.randn(5, 4, dtype=torch.float64, requires_grad=True), torch.randn(7, 4, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([6, 0, -100, 3, 3])
    assert torch.autograd.gradcheck(lambda a, b: ab.token_losses(a, b, t), (h, w))
    assert torch.autograd.gradgradcheck(lambda a, b: ab.token_losses(a, b, t), (h, w))
    got = torch.func.vmap(lambda a: ab.token_losses(a, w, t))(torch.stack((h, 2 * h)))
    assert torch.allclose(got[1], ab.token_losses(2 * h, w, t))


def test_token_losses_in_torch_operations_twice():
    """The function that a backward pass takes which is differentiated in turn."""
    gen = torch.Generator().manual_seed(2)
    h, w, g = (torch.randn(*s, generator=gen, dtype=torch.float64, requires_grad=True) for s in ((6, 4), (9, 4), (6,)))
    t = torch.tensor([8, 0, -100, 3, 3, 1])
    want = torch.autograd.grad(ab.token_losses(h, w, t), (h, w), g)
    got = BACKWARD["token_losses"](g, h, w, t, -100, True, True)
    assert torch.allclose(got[0], want[0]) and torch.allclose(got[1], want[1])
    assert torch.autograd.gradcheck(lambda *a: BACKWARD["token_losses"](*a, t, -100, True, True)[:2], (g, h, w))
    assert BACKWARD["token_losses"](g, h, w, t, -100, False, True)[0] is None


def test_rows_that_are_not_scored_reach_nothing():
    h, w = torch.randn(4, 6), torch.randn(5, 6, requires_grad=True)
    t = torch.tensor([1, -100, 4, -100])
    h[1], h[3] = torch.nan, torch.inf
    h.requires_grad_()
    loss = ab.token_losses(h, w, t)
    dh, dw = torch.autograd.grad(loss.sum(), (h, w))
    assert not loss[[1, 3]].any() and not dh[[1, 3]].any() and dw.isfinite().all() and dh.isfinite().all()
    outside = ab.token_losses(h, w, torch.tensor([5, -100, -1, -100]))
    assert torch.equal(outside.isnan(), torch.tensor([True, False, True, False]))


def test_token_losses_refusals():
    h, w, t = torch.randn(3, 4), torch.randn(5, 4), torch.tensor([1, 2, 0])
    for call, words in (
            (lambda: ab.token_losses(h, w.t(), t), r"hidden \[..., size\] and weight \[vocab, size\]"),
            (lambda: ab.token_losses(h, w[0], t), r"weight \[vocab, size\]"),
            (lambda: ab.token_losses(h, w[:0], t), "not empty"),
            (lambda: ab.token_losses(torch.tensor(1.0), w, t), r"hidden \[..., size\]"),
            (lambda: ab.token_losses(h, w, t[:2]), r"targets must be int64 or int32 \(3,\)"),
            (lambda: ab.token_losses(h, w, t.float()), "targets must be int64 or int32"),
            (lambda: ab.token_losses(h, w.bfloat16(), t), "one floating-point type"),
            (lambda: ab.token_losses(h.long(), w.long(), t), "one floating-point type"),
            (lambda: ab.token_losses(h, w, t, 1.5), "ignore_index must be an int"),
            (lambda: ab.token_losses(h, w, t, True), "ignore_index must be an int")):
        with pytest.raises(ValueError, match=words):
            call()


def test_token_losses_entry_points():
    lib = _hip.open_library()
    f32, bf16 = _hip.DT_F32, _hip.DT_BF16
    fwd, back = lib.adambridge_token_losses, lib.adambridge_token_losses_backward
    work, back_work = lib.adambridge_token_losses_work, lib.adambridge_token_losses_backward_work
    for dtype, sizes in ((f32, (0, 8, 8)), (f32, ((1 << 23) + 1, 8, 8)), (f32, (4, 0, 8)), (f32, (4, (1 << 22) + 1, 8)), (f32, (4, 8, 3)),
                         (bf16, (4, 8, 7)), (bf16, (4, 8, (1 << 20) + 1))):
        assert fwd(P, P, dtype, P, *sizes, -100, P, P, P) == EBADN and work(dtype, *sizes) == EBADN
        assert back(P, P, P, dtype, P, *sizes, -100, P, P, P, P) == EBADN and back_work(dtype, *sizes) == EBADN
    assert fwd(P, P, _hip.DT_FP8, P, 4, 8, 8, -100, P, P, P) == EDTYPE and work(_hip.DT_FP8, 4, 8, 8) == EDTYPE
    assert back(P, P, P, 9, P, 4, 8, 8, -100, P, P, P, P) == EDTYPE and back_work(9, 4, 8, 8) == EDTYPE
    for i in (0, 1, 3, 8, 10):
        args = [P, P, f32, P, 4, 8, 8, -100, P, P, P]
        args[i] = None
        assert fwd(*args) == ENULL
    for i in (0, 1, 2, 4, 9, 12):
        args = [P, P, P, f32, P, 4, 8, 8, -100, P, P, P, P]
        args[i] = None
        assert back(*args) == ENULL
    assert fwd(P, P, f32, P, 4, 8, 8, -100, P, P, ctypes.c_void_p(264)) == EALIGN
    assert back(P, P, P, f32, P, 4, 8, 8, -100, P, P, P, ctypes.c_void_p(264)) == EALIGN
    assert back(P, P, P, f32, P, 4, 8, 8, -100, P, None, None, P) == 0   # nothing wanted
    # half a GiB of a piece's gradient, or 4096 words for every row
    assert back_work(bf16, 16384, 151936, 8) < 3 << 28 and back_work(bf16, 1 << 20, 151936, 8) < (1 << 20) * 4352 * 2 + (1 << 27)
