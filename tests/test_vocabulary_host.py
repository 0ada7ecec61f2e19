"""A language model's ends on the CPU: torch operations of the same values, what the calls and the C entry points refuse."""

import ctypes

import pytest
import torch

import adambridge_amd as ab
from adambridge_amd import _hip

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
    assert lib.adambridge_embed_work(64, 4, 4) == 64 * 8 and lib.adambridge_embed_work(65, 4, 4) == 65 * 8 + 2 * 2 * 4 * 4
