"""The expert block's operators in torch operations, on the CPU: operands at the edge of what they take."""

import ctypes

import pytest
import torch

import adambridge_amd as ab
from adambridge_amd import _hip


def test_decreasing_ends_share_no_rows():
    """An end below one before it counts as that: each row is one expert's, and the result has the rows of x."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(9, 4, generator=gen, dtype=torch.float64, requires_grad=True)
    w = torch.randn(5, 3, 4, generator=gen, dtype=torch.float64, requires_grad=True)
    g = torch.randn(9, 3, generator=gen, dtype=torch.float64)
    for ends, same in (([5, 3, 8, 2, 9], [5, 5, 8, 8, 9]), ([-2, 4, 1, 1, 6], [0, 4, 4, 4, 6]), ([12, 3, 3, 20, 1], [9] * 5)):
        out, want = (ab.expert_mm(x, w, torch.tensor(e, dtype=torch.int32)) for e in (ends, same))
        assert out.shape == (9, 3) and torch.equal(out, want)
        for a, b in zip(torch.autograd.grad(out, (x, w), g), torch.autograd.grad(want, (x, w), g)):
            assert torch.equal(a, b)


def test_autocast_casts_what_a_linear_s_does():
    """float32 and half types; float64 stays, whole numbers and a float64 beside a float32 are refused."""
    x, w, ends = torch.randn(6, 4, dtype=torch.float64), torch.randn(2, 3, 4, dtype=torch.float64), torch.tensor([2, 6], dtype=torch.int32)
    want = ab.expert_mm(x, w, ends)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert torch.equal(ab.expert_mm(x, w, ends), want)
        assert ab.expert_mm(x.float(), w.float(), ends).dtype == torch.bfloat16
        assert ab.expert_mm(x.half(), w.float(), ends).dtype == torch.bfloat16
        for a, b in ((x.long(), w.float()), (x.long(), w.long()), (x.float(), w)):
            with pytest.raises(ValueError, match="one floating-point type"):
                ab.expert_mm(a, b, ends)


def test_positions_outside_the_rows_count_as_zeros():
    """As in the kernels: no error of an index, on whatever device."""
    gen = torch.Generator().manual_seed(3)
    r = ab.route(torch.randn(5, 4, generator=gen), 2)
    position = r.position.clone()
    position[1, 1], position[3, 0] = 10, -1
    bad, keep = r._replace(position=position), torch.ones(5, 2)
    keep[1, 1] = keep[3, 0] = 0.0
    y = torch.randn(10, 6, generator=gen, requires_grad=True)
    weights = r.weights.clone().requires_grad_()
    out, want = ab.combine(y, bad._replace(weights=weights)), ab.combine(y, r._replace(weights=weights * keep))
    assert torch.allclose(out, want)
    g = torch.randn(5, 6, generator=gen)
    for a, b in zip(torch.autograd.grad(out, (y, weights), g), torch.autograd.grad(want, (y, weights), g)):
        assert torch.allclose(a, b)
    x = torch.randn(5, 6, generator=gen, requires_grad=True)
    rows = ab.dispatch(x, bad)
    named = position[(position >= 0) & (position < 10)].long()
    assert torch.equal(rows[named], ab.dispatch(x, r)[named])
    g = torch.zeros(10, 6)
    g[named] = 1.0
    assert torch.equal(torch.autograd.grad(rows, x, g)[0], keep.sum(1, keepdim=True).expand(5, 6))


def test_scratch_of_a_norm_s_gradient_is_at_a_word():
    """Refused before anything is launched."""
    lib, p = _hip.open_library(), ctypes.c_void_p(256)
    for offset in (1, 2, 3):
        rc = lib.adambridge_layer_norm_backward(p, p, _hip.DT_F32, None, _hip.DT_F32, p, 4, 4, p, p, p, ctypes.c_void_p(256 + offset))
        assert rc == -14


def test_routings_of_a_batch():
    """vmap over logits gives each one's routing, and what is dispatched and combined by it."""
    gen = torch.Generator().manual_seed(5)
    logits, x, y = (torch.randn(3, *s, generator=gen) for s in ((6, 4), (6, 5), (12, 5)))
    for normalize in (True, False):
        one_by_one = [ab.route(t, 2, normalize) for t in logits]
        at_once = torch.func.vmap(lambda t: tuple(ab.route(t, 2, normalize)))(logits)
        for i, got in enumerate(at_once):
            assert torch.equal(got, torch.stack([r[i] for r in one_by_one]))
    one_by_one = [ab.route(t, 2) for t in logits]
    got = torch.func.vmap(lambda t, a: ab.dispatch(a, ab.route(t, 2)))(logits, x)
    assert torch.equal(got, torch.stack([ab.dispatch(a, r) for a, r in zip(x, one_by_one)]))
    got = torch.func.vmap(lambda t, a: ab.combine(a, ab.route(t, 2)))(logits, y)
    assert torch.allclose(got, torch.stack([ab.combine(a, r) for a, r in zip(y, one_by_one)]))
