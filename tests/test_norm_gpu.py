"""layer_norm by the library's kernels (csrc/abh_norm.hip) against its definition in 64 bits."""

import pytest
import torch

import adambridge_amd as ab
from adambridge_amd import _hip, norms

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -23}   # twice the half ulp a rounding costs


def _case(rows, cols, dtype, w_dtype, seed=0, shift=0.4):
    gen = torch.Generator("cuda").manual_seed(seed)
    x = (torch.randn(rows, cols, generator=gen, device="cuda") * 2.0 + shift).to(dtype)
    w = b = None
    if w_dtype is not None:
        w = (torch.randn(cols, generator=gen, device="cuda") * 0.5 + 1.0).to(w_dtype)
        b = torch.randn(cols, generator=gen, device="cuda").to(w_dtype)
    g = torch.randn(rows, cols, generator=gen, device="cuda").to(dtype)
    return x, w, b, g


def _check(x, w, b, g, eps=1e-5):
    leaves = [t if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = ab.layer_norm(*leaves, eps)
    given = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, given, g)
    with torch.no_grad():
        assert torch.equal(ab.layer_norm(x, w, b, eps), y)   # the call without a gradient is the same kernel
    assert y.dtype == x.dtype and [d.dtype for d in grads] == [t.dtype for t in given]
    xd, gd = x.double(), g.double()
    wd = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda") if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    var, mean = torch.var_mean(xd, -1, correction=0, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = (xd - mean) * rstd
    # FP32 inside: the mean is off by some roundings (a tree's, below 2^5 of them) of the row's largest value, and
    # everything after it by a few of its own size: 2^-24 2^6 of max|x| rstd and of the terms
    lost = 2.0 ** -18 * (1.0 + xd.abs().amax(-1, keepdim=True) * rstd)
    want = xh * wd + bd
    unit = UNIT[x.dtype]
    assert ((y.double() - want).abs() <= want.abs() * unit + lost * (wd.abs() * (1.0 + xh.abs())) + 1e-30).all()
    gw = gd * wd
    c1, c2 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
    dx = rstd * (gw - c1 - xh * c2)
    size = rstd * (gw.abs() + gw.abs().mean(-1, keepdim=True) + xh.abs() * (gw * xh).abs().mean(-1, keepdim=True) + gw.abs())
    assert ((grads[0].double() - dx).abs() <= dx.abs() * unit + lost * size * (1.0 + xh.abs()) + 1e-30).all()
    flat = (gd * xh).reshape(-1, x.shape[-1])
    if w is not None:
        wunit = UNIT[w.dtype]
        dw, slack = flat.sum(0), (lost * (1.0 + xh.abs()) * gd.abs()).reshape(flat.shape).sum(0)
        assert ((grads[1].double() - dw).abs() <= dw.abs() * wunit + slack + flat.abs().sum(0) * 2.0 ** -18).all()
    if b is not None:
        wunit = UNIT[b.dtype]
        db = gd.reshape(flat.shape).sum(0)
        assert ((grads[-1].double() - db).abs() <= db.abs() * wunit + gd.reshape(flat.shape).abs().sum(0) * 2.0 ** -18).all()


# one value; less than a vector; rows off the 16-byte boundary; every number of lanes and vectors a row, at its
# ends; rows beyond the registers (backward from 16385 BF16 values, forward from 32769; half of it in FP32)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (2, 255), (70, 513), (9, 1024), (33, 1025), (130, 2048), (3, 2049),
                                       (2, 4099), (3, 8192), (2, 8193), (3, 16385), (2, 32771), (1, 40000), (1030, 96), (2060, 2051)])
def test_matches_the_definition(rows, cols, dtype):
    _check(*_case(rows, cols, dtype, dtype, seed=rows + cols))


@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, None),
                                           (torch.bfloat16, None)])
@pytest.mark.parametrize("rows,cols", [(37, 333), (5, 4100), (2, 20011)])
def test_weights_of_another_type_or_none(rows, cols, dtype, w_dtype):
    _check(*_case(rows, cols, dtype, w_dtype))


def test_weight_or_bias_alone():
    x, w, b, g = _case(19, 260, torch.bfloat16, torch.bfloat16)
    _check(x, w, None, g)
    _check(x, None, b, g)


def test_large_mean_and_constant_rows():
    """The variance is the mean of squared deviations: a mean of 1000 times the deviation costs no more than the
    mean's own rounding; a constant row gives the bias and finite gradients."""
    _check(*_case(12, 1000, torch.float32, torch.float32, shift=2000.0))
    x, w, b, g = _case(4, 640, torch.bfloat16, torch.bfloat16)
    x[1] = 3.0
    leaf = x.requires_grad_()
    y = ab.layer_norm(leaf, w, b)
    assert torch.equal(y[1], b)
    assert torch.isfinite(torch.autograd.grad(y, leaf, g)[0]).all()


def test_infinities_and_nan_stay_in_their_rows():
    x, w, b, g = _case(6, 700, torch.float32, torch.float32)
    clean = ab.layer_norm(x, w, b)
    x[1, 5], x[4, 699] = torch.nan, torch.inf
    y = ab.layer_norm(x, w, b)
    assert y[1].isnan().all() and y[4].isnan().all()
    keep = [0, 2, 3, 5]
    assert torch.equal(y[keep], clean[keep])


def test_shapes_strides_and_empty_batches():
    x, w, b, g = _case(24, 96, torch.bfloat16, torch.bfloat16)
    want = ab.layer_norm(x, w, b)
    assert torch.equal(ab.layer_norm(x.view(2, 3, 4, 96), w, b), want.view(2, 3, 4, 96))
    wide = torch.zeros(24, 200, dtype=x.dtype, device="cuda")
    wide[:, 3:99] = x
    leaf = wide.requires_grad_()
    y = ab.layer_norm(leaf[:, 3:99], w, b)
    assert torch.equal(y, want)
    dx, = torch.autograd.grad(y, leaf, g.t().contiguous().t())
    assert not dx[:, :3].any() and not dx[:, 99:].any() and dx[:, 3:99].any()
    assert ab.layer_norm(x[:0], w, b).shape == (0, 96)


def test_gradient_against_differences():
    x, w, b, g = _case(5, 300, torch.float32, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ab.layer_norm(*leaves), leaves, g)
    gen = torch.Generator("cuda").manual_seed(5)
    with torch.no_grad():
        for i in range(3):
            d = torch.randn(leaves[i].shape, generator=gen, device="cuda")
            h = 2.0 ** -7
            at = [[t + s * h * d if j == i else t for j, t in enumerate(leaves)] for s in (1, -1)]
            up, down = (((ab.layer_norm(*a).double()) * g.double()).sum() for a in at)
            want = (grads[i].double() * d.double()).sum()
            # the outputs are below 16 and rounded to 2^-20: 1500 of them times g, over 2 h; and the third
            # derivative's h^2 of the sum's size
            assert abs((up - down) / (2 * h) - want) <= 1500 ** 0.5 * 4 * 2.0 ** -20 / h + 1500 ** 0.5 * 8 * h ** 2


def test_only_the_wanted_gradients_and_the_second_derivative():
    x, w, b, g = _case(11, 130, torch.float32, torch.float32)
    for i in range(3):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        all_leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        one, = torch.autograd.grad(ab.layer_norm(*leaves), leaves[i], g)
        assert torch.equal(one, torch.autograd.grad(ab.layer_norm(*all_leaves), all_leaves, g)[i])
    small = [t[..., :6].double().cpu().float() for t in (x, w, b)]
    # differentiated twice: the gradient of a gradient's sum, kernels forward, torch operations backward
    got, want = [], []
    for out, device in ((got, "cuda"), (want, "cpu")):
        leaves = [t.to(device).requires_grad_() for t in small]
        dx, = torch.autograd.grad((ab.layer_norm(*leaves) * g[:, :6].to(device)).sum(), leaves[0], create_graph=True)
        out += [t.cpu() for t in torch.autograd.grad(dx.square().sum(), leaves[:2])]
    for a, c in zip(got, want):
        assert torch.allclose(a, c, rtol=1e-3, atol=1e-3)


def test_the_kernels_run_and_refuse_wrong_operands(monkeypatch):
    x, w, b, g = _case(4, 64, torch.bfloat16, torch.bfloat16)
    k = _hip.load()
    with pytest.raises(ValueError, match="x must be contiguous"):
        k.layer_norm(x.t(), None, None, 1e-5, False)
    with pytest.raises(ValueError, match="weight must be contiguous"):
        k.layer_norm(x, w[:10], b, 1e-5, False)
    with pytest.raises(ValueError, match="bias must be contiguous"):
        k.layer_norm(x, w, b.float(), 1e-5, False)
    with pytest.raises(ValueError, match="gout must be contiguous"):
        k.layer_norm_backward(g.float(), x, w, torch.empty(4, 2, device="cuda"), w.dtype, (True, True, True))
    monkeypatch.setattr(norms, "_torch_layer_norm", None)   # the ordinary call does not come here
    ab.layer_norm(x, w, b)
