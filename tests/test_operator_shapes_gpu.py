"""Layer norm, dispatch and combine at sizes whose launches the smaller ones do not reach."""

import pytest
import torch

import adambridge_amd as ab
from test_norm_gpu import UNIT, _case, _check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


# from 2048 rows on, 2048, 8192 and 16384 columns are on fewer lanes than with fewer rows
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(2051, 2048), (2048, 1999), (2050, 8192), (2049, 5003), (2048, 16384), (2053, 9001)])
def test_many_rows_of_wide_norms(rows, cols, dtype):
    _check(*_case(rows, cols, dtype, dtype, seed=cols))


# x of more than 128 MB: streamed in the backward pass, at each of its numbers of lanes a row
@pytest.mark.parametrize("rows,cols,dtype", [(300001, 230, torch.bfloat16), (140003, 500, torch.bfloat16), (70001, 1000, torch.bfloat16),
                                             (35003, 1999, torch.bfloat16), (16500, 4096, torch.bfloat16), (8501, 8191, torch.bfloat16),
                                             (4200, 16384, torch.bfloat16), (70003, 500, torch.float32), (9001, 4000, torch.float32)])
def test_streamed_norm_gradients(rows, cols, dtype):
    _check(*_case(rows, cols, dtype, dtype, seed=cols))


# from 4096 tokens on a wavefront takes several vectors of a row; the last two are more than one wavefront's
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,k,hidden", [(4096, 2, 1024), (4099, 3, 1501), (4100, 2, 4609), (5001, 1, 8200)])
def test_many_tokens_of_several_vectors(tokens, k, hidden, dtype):
    gen = torch.Generator("cuda").manual_seed(hidden)
    r = ab.route(torch.randn(tokens, 16, generator=gen, device="cuda"), k)
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype).requires_grad_()
    rows = ab.dispatch(x, r)
    token = r.order.long() // k
    assert torch.equal(rows, x[token])
    y = torch.randn(tokens * k, hidden, generator=gen, device="cuda").to(dtype).requires_grad_()
    weights = r.weights.clone().requires_grad_()
    out = ab.combine(y, r._replace(weights=weights))
    grows, gout = (torch.randn(*t.shape, generator=gen, device="cuda").to(dtype) for t in (rows, out))
    dx, = torch.autograd.grad(rows, x, grows)
    dy, dw = torch.autograd.grad(out, (y, weights), gout)

    def summed(got, terms):   # k terms in FP32, one rounding
        want = terms.sum(1)
        assert ((got.double() - want).abs() <= want.abs() * UNIT[dtype] + terms.abs().sum(1) * k * 2.0 ** -23).all()

    place = r.position.long()
    summed(dx, grows.double()[place])
    summed(out, y.detach().double()[place] * r.weights.double()[:, :, None])
    want = r.weights.double().reshape(-1)[r.order.long()][:, None] * gout.double()[token]
    assert ((dy.double() - want).abs() <= want.abs() * UNIT[dtype]).all()
    products = y.detach().double()[place] * gout.double()[:, None, :]
    assert ((dw.double() - products.sum(2)).abs() <= products.abs().sum(2) * (hidden / 64 + 16) * 2.0 ** -23).all()
