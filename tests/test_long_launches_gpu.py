"""Calls of so many rows that their launches have 2^32 lanes and more, which one dimension of a grid does not hold."""

import pytest
import torch

import adambridge_amd as ab

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def _ends_of(t, count=4099):
    """The first and last rows of ``t`` and those around the middle."""
    half = t.shape[0] // 2
    return torch.cat((t[:count], t[half:half + count], t[-count:]))


def test_layer_norm_of_more_rows_than_a_grid_holds():
    rows = (1 << 29) + 8195
    x = torch.randint(-9, 9, (rows, 2), device="cuda", dtype=torch.int8).bfloat16().requires_grad_()
    weight = torch.tensor([0.5, 2.0], device="cuda", dtype=torch.bfloat16)
    bias = torch.tensor([1.0, -1.0], device="cuda", dtype=torch.bfloat16)
    y = ab.layer_norm(x, weight, bias)
    some = _ends_of(x.detach()).double().requires_grad_()
    want = torch.nn.functional.layer_norm(some, (2,), weight.double(), bias.double())
    assert ((_ends_of(y.detach()).double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -18).all()
    g = torch.ones_like(y)
    grad, = torch.autograd.grad(y, x, g)
    want_grad, = torch.autograd.grad(want, some, torch.ones_like(want))
    # g w = (0.5, 2) less its mean and its part along xh: a difference of numbers of size up to 2 rstd
    rstd = (some.detach().var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    assert ((_ends_of(grad).double() - want_grad).abs() <= want_grad.abs() * 2.0 ** -8 + rstd * 2.0 ** -18).all()


def test_routing_of_more_tokens_than_a_grid_holds():
    tokens, n, cols = (1 << 28) + 77, 3, 2
    logits = torch.randint(-9, 9, (tokens, n), device="cuda", dtype=torch.int8).bfloat16().requires_grad_()
    r = ab.route(logits, 1, normalize=False)
    best = logits.detach().max(1)
    first = (logits.detach() == best.values[:, None]).int().argmax(1)   # the lowest of equal ones
    assert torch.equal(r.experts[:, 0].long(), first)
    counts = torch.bincount(first, minlength=n)
    assert torch.equal(r.ends.long(), counts.cumsum(0))
    start = 0
    for e in range(n):   # stable: an expert's rows in the tokens' order
        mine = torch.nonzero(first == e).flatten()
        assert torch.equal(r.order[start:start + mine.numel()].long(), mine)
        assert torch.equal(r.position[mine, 0].long(), torch.arange(start, start + mine.numel(), device="cuda"))
        start += mine.numel()
        del mine
    del first, best, counts
    some = _ends_of(logits.detach()).double().requires_grad_()
    want = some.softmax(1).max(1, keepdim=True).values
    assert ((_ends_of(r.weights.detach()).double() - want).abs() <= 2.0 ** -20).all()
    grad, = torch.autograd.grad(r.weights, logits, torch.ones_like(r.weights))
    chosen = _ends_of(r.experts).long()
    want_grad, = torch.autograd.grad(some.softmax(1).gather(1, chosen).sum(), some)
    assert ((_ends_of(grad).double() - want_grad).abs() <= want_grad.abs() * 2.0 ** -8 + 2.0 ** -20).all()
    del grad, chosen

    r = ab.Routing(r.weights.detach(), *r[1:])
    x = torch.randint(-99, 99, (tokens, cols), device="cuda", dtype=torch.int8).bfloat16()
    rows = ab.dispatch(x, r)
    assert torch.equal(rows, x[r.order.long()])
    rows.requires_grad_()
    weights = r.weights.clone().requires_grad_()
    y = ab.combine(rows, r._replace(weights=weights))
    assert torch.equal(y.detach(), (weights.detach() * x.float()).bfloat16())   # one choice: a product, rounded once
    drows, dweights = torch.autograd.grad(y, (rows, weights), x)
    assert torch.equal(drows[r.position[:, 0].long()], (weights.detach() * x.float()).bfloat16())
    assert torch.equal(dweights, x.float().square().sum(1, keepdim=True))       # whole numbers: exact


@pytest.mark.parametrize("n,k", [(1 << 16, 2), (1, 1 << 19)])
def test_expert_mm_of_more_tiles_than_a_grid_holds(n, k):
    experts = 4096                     # a row each, and one that is no expert's
    x = torch.randint(-9, 9, (experts + 1, k), device="cuda", dtype=torch.int8).bfloat16().requires_grad_()
    weight = torch.empty(experts, n, k, device="cuda", dtype=torch.bfloat16).random_(-9, 9)
    ends = torch.arange(1, experts + 1, device="cuda", dtype=torch.int32)
    y = ab.expert_mm(x, weight, ends)
    g = torch.randint(-9, 9, y.shape, device="cuda", dtype=torch.int8).bfloat16()
    dx, = torch.autograd.grad(y, x, g)
    assert not y[-1].any() and not dx[-1].any()
    for e in range(0, experts, 128):   # whole numbers, so exact but for the one rounding (2^23 at most: FP32 holds them)
        w, some = weight[e:e + 128].double(), slice(e, e + 128)
        assert torch.equal(y[some], (w * x.detach()[some, None].double()).sum(2).bfloat16())
        assert torch.equal(dx[some], (w * g[some, :, None].double()).sum(1).bfloat16())
