"""The expert layer and layer norm on the CPU: torch operations of the same values, and what the calls refuse."""

import ctypes

import pytest
import torch

import adambridge_amd as ab
from adambridge_amd import _hip


def test_layer_norm_is_torch_s():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(4, 5, 12, generator=gen, requires_grad=True)
    norm = torch.nn.LayerNorm(12)
    y, want = ab.layer_norm(x, norm.weight, norm.bias, norm.eps), norm(x)
    assert torch.allclose(y, want, rtol=1e-6, atol=1e-6)
    g = torch.randn(4, 5, 12, generator=gen)
    for a, b in zip(torch.autograd.grad(y, (x, norm.weight), g), torch.autograd.grad(want, (x, norm.weight), g)):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    assert ab.layer_norm(x.bfloat16(), norm.weight).dtype == torch.bfloat16


def test_a_block_is_the_loop_over_tokens():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(9, 16, generator=gen, dtype=torch.float64)
    gate, up, down = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((5, 16), (5, 24, 16), (5, 16, 24)))
    r = ab.route(x @ gate.t(), 2)
    y = ab.combine(ab.expert_mm(ab.expert_mm(ab.dispatch(x, r), up, r.ends).relu(), down, r.ends), r)
    for t in range(9):
        weights, chosen = torch.topk(x[t] @ gate.t(), 2)
        want = sum(w * (down[e] @ (up[e] @ x[t]).relu()) for w, e in zip(torch.softmax(weights, 0), chosen))
        assert torch.equal(r.experts[t].long(), chosen)
        assert torch.allclose(y[t], want, rtol=1e-6, atol=1e-8)   # the weights are FP32
    assert r.ends[-1] == 18 and torch.equal(r.position.reshape(-1)[r.order.long()].long(), torch.arange(18))


def test_gradients_on_the_cpu():
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(7, 6, generator=gen, dtype=torch.float64, requires_grad=True)
    w = torch.randn(3, 4, 6, generator=gen, dtype=torch.float64, requires_grad=True)
    ends = torch.tensor([2, 2, 5], dtype=torch.int32)
    assert torch.autograd.gradcheck(lambda a, b: ab.expert_mm(a, b, ends), (x, w))
    r = ab.route(torch.randn(7, 4, generator=gen), 2)
    assert torch.autograd.gradcheck(lambda a: ab.dispatch(a, r), (x,))
    rows = torch.randn(14, 6, generator=gen, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a: ab.combine(a, r), (rows,))


def test_masked_rows_have_no_weight_and_no_gradient():
    logits = torch.full((2, 4), -torch.inf)
    logits[1, 2] = 0.5
    leaf = logits.requires_grad_()
    for normalize in (True, False):
        r = ab.route(leaf, 3, normalize=normalize)
        assert not r.weights[0].any() and torch.equal(r.weights[1], torch.tensor([1.0, 0.0, 0.0]))
        assert torch.equal(r.experts[1], torch.tensor([2, 0, 1], dtype=torch.int32))


def test_refusals():
    x, w = torch.randn(6, 16), torch.randn(2, 8, 16)
    ends = torch.tensor([2, 6], dtype=torch.int32)
    r = ab.route(torch.randn(6, 4), 2)
    for call, words in (
            (lambda: ab.layer_norm(torch.tensor(1.0)), "rows of one value or more"),
            (lambda: ab.layer_norm(torch.ones(3, 4, dtype=torch.int32)), "floating-point rows"),
            (lambda: ab.layer_norm(x, torch.ones(8)), r"weight must be \[16\]"),
            (lambda: ab.layer_norm(x, torch.ones(16), torch.ones(16).bfloat16()), "of one type"),
            (lambda: ab.route(torch.randn(3), 1), r"\[tokens, experts\]"),
            (lambda: ab.route(torch.randn(3, 4), 5), "top_k must be an int"),
            (lambda: ab.route(torch.randn(3, 4), 0), "top_k must be an int"),
            (lambda: ab.route(torch.randn(3, 4), True), "top_k must be an int"),
            (lambda: ab.route(torch.ones(3, 4).long(), 1), "floating-point"),
            (lambda: ab.dispatch(x[:5], r), "5 tokens, the routing 6"),
            (lambda: ab.dispatch(x, r._replace(position=r.position.long())), "int32"),
            (lambda: ab.combine(x, r), "the routing's 12, got 6"),
            (lambda: ab.combine(torch.randn(12, 4), r._replace(weights=r.weights.double())), "weights must be float32"),
            (lambda: ab.expert_mm(x, w.transpose(1, 2), ends), r"x \[rows, in\]"),
            (lambda: ab.expert_mm(x, w, ends[:1]), "ends must be int32"),
            (lambda: ab.expert_mm(x, w, ends.long()), "ends must be int32"),
            (lambda: ab.expert_mm(x, w.bfloat16(), ends), "one floating-point type"),
            (lambda: ab.expert_mm(x[:, :0], w[:, :, :0], ends), "must not be empty")):
        with pytest.raises(ValueError, match=words):
            call()


def test_entry_points_check_sizes_types_and_addresses():
    """The C entry points' codes, without a device: nothing is launched for a refused call."""
    lib = _hip.open_library()
    f32, bf16, p = _hip.DT_F32, _hip.DT_BF16, ctypes.c_void_p(256)
    ebadn, enull, edtype, ealign = -1, -2, -4, -14
    norm, back = lib.adambridge_layer_norm, lib.adambridge_layer_norm_backward
    assert norm(p, f32, None, None, f32, 0, 4, 1e-5, p, None) == ebadn
    assert norm(p, f32, None, None, f32, 4, (1 << 30) + 1, 1e-5, p, None) == ebadn
    assert norm(p, _hip.DT_FP8, None, None, f32, 4, 4, 1e-5, p, None) == edtype
    assert norm(p, f32, None, None, _hip.DT_NONE, 4, 4, 1e-5, p, None) == edtype
    assert norm(None, f32, None, None, f32, 4, 4, 1e-5, p, None) == enull
    assert back(p, p, f32, None, f32, None, 4, 4, p, None, None, None) == enull
    assert back(p, p, f32, None, f32, p, 4, 4, p, p, None, None) == enull   # a weight's gradient without work
    assert back(p, p, f32, None, f32, p, 4, 4, None, None, None, None) == 0
    assert lib.adambridge_layer_norm_work(0, 4, f32) == ebadn and lib.adambridge_layer_norm_work(4, 4, 9) == edtype
    assert lib.adambridge_layer_norm_work(8, 100, bf16) % 800 == 0

    assert lib.adambridge_route_work(64, 8, 2) == 0 and lib.adambridge_route_work(65, 8, 2) > 0
    for sizes in ((0, 8, 2), (8, 1025, 2), (8, 8, 9), (8, 100, 65), (8, 8, 0), (1 << 30, 8, 4)):
        assert lib.adambridge_route_work(*sizes) == ebadn
        assert lib.adambridge_route(p, f32, *sizes, 1, p, p, p, p, p, p) == ebadn
        assert lib.adambridge_route_backward(p, p, p, p, f32, *sizes, 1, p) == ebadn
    assert lib.adambridge_route(p, 7, 8, 8, 2, 1, p, p, p, p, p, p) == edtype
    assert lib.adambridge_route(p, f32, 65, 8, 2, 1, p, p, p, p, p, None) == enull
    assert lib.adambridge_route(p, f32, 65, 8, 2, 1, p, p, p, p, p, ctypes.c_void_p(258)) == ealign
    assert lib.adambridge_route_backward(p, p, p, None, f32, 8, 8, 2, 0, p) == enull

    assert lib.adambridge_dispatch(p, f32, p, 8, 65, 8, p) == ebadn and lib.adambridge_dispatch(p, f32, p, 8, 2, 0, p) == ebadn
    assert lib.adambridge_dispatch(p, 0, p, 8, 2, 8, p) == edtype and lib.adambridge_dispatch(p, f32, None, 8, 2, 8, p) == enull
    assert lib.adambridge_combine(None, f32, None, p, 8, 2, 8, p) == enull
    assert lib.adambridge_combine_backward(p, None, f32, p, p, 8, 2, 8, p, p) == enull
    assert lib.adambridge_combine_backward(p, None, f32, p, p, 8, 2, 8, None, None) == 0

    size = lib.adambridge_expert_mm_work
    for product, fn in enumerate((lib.adambridge_expert_mm, lib.adambridge_expert_mm_dx, lib.adambridge_expert_mm_dw)):
        for sizes in ((-1, 2, 8, 8), ((1 << 30) + 1, 2, 8, 8), (4, 0, 8, 8), (4, 4097, 8, 8), (4, 2, 0, 8), (4, 2, 8, (1 << 22) + 1)):
            assert fn(p, p, p, p, f32, *sizes, p) == ebadn and size(product, f32, *sizes) == ebadn
        assert fn(p, p, p, p, _hip.DT_F24, 4, 2, 8, 8, p) == edtype and size(product, _hip.DT_F24, 4, 2, 8, 8) == edtype
        assert fn(p, p, None, p, f32, 4, 2, 8, 8, p) == enull and fn(p, None, p, p, f32, 4, 2, 8, 8, p) == enull
        assert size(product, bf16, 4, 2, 8, 8) == 0
    assert size(3, f32, 4, 2, 8, 8) == ebadn
    assert size(2, bf16, 9000, 1, 64, 64) > 0 and size(1, bf16, 8192, 8, 8192, 2048) > 0
    assert lib.adambridge_expert_mm_dw(p, p, p, p, bf16, 9000, 1, 64, 64, None) == enull
    assert lib.adambridge_expert_mm_dw(p, p, p, p, bf16, 9000, 1, 64, 64, ctypes.c_void_p(264)) == ealign
    assert lib.adambridge_expert_mm(None, p, p, None, f32, 0, 2, 8, 8, None) == 0   # no rows: nothing to do
