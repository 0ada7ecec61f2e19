"""The operators' C entry points between guards: operands inside a buffer of NaN, at any element's address, results inside
one of a value that no call writes.  A value read from outside an operand shows in the result, one written outside a result
in its guard (all of it inside allocations of the test's own)."""

import pytest
import torch

import adambridge_amd as ab
from adambridge_amd import _hip

pytestmark = pytest.mark.gpu
GUARD = 4096        # values on either side
MARK = 24576.0      # exact in both types
CODES = {torch.float32: _hip.DT_F32, torch.bfloat16: _hip.DT_BF16}


def _inside(t, shift):
    """``t`` in a buffer of NaN (whole numbers: of their largest), ``shift`` values after a 16-byte boundary."""
    guard = float("nan") if t.is_floating_point() else torch.iinfo(t.dtype).max
    whole = torch.full((t.numel() + 2 * GUARD + 8,), guard, dtype=t.dtype, device="cuda")
    part = whole[GUARD + shift:GUARD + shift + t.numel()].view(t.shape)
    part.copy_(t)
    return part


class _Result:
    def __init__(self, shape, dtype, shift):
        self.n = torch.Size(shape).numel()
        self.mark = MARK if dtype.is_floating_point else -7
        self.whole = torch.full((self.n + 2 * GUARD + 8,), self.mark, dtype=dtype, device="cuda")
        self.lo = GUARD + shift
        self.value = self.whole[self.lo:self.lo + self.n].view(shape)

    def check(self, want, close=None):
        assert (self.whole[:self.lo] == self.mark).all() and (self.whole[self.lo + self.n:] == self.mark).all()
        assert torch.equal(self.value, want) if close is None else torch.allclose(self.value, want, **close)


def _call(name, *args):
    lib = _hip.load()
    lib.set_stream(torch.cuda.current_stream())
    rc = getattr(lib._lib, name)(*[a.value.data_ptr() if isinstance(a, _Result) else a.data_ptr() if isinstance(a, torch.Tensor) else a
                                   for a in args])
    assert rc == 0, (name, rc)


def _work(name, *sizes):
    nbytes = getattr(_hip.load()._lib, name)(*sizes)
    assert nbytes >= 0
    return _Result(((nbytes + 3) // 4,), torch.int32, 0) if nbytes else None


# streamed, small, large (a cut rest) and FP32 tiles, sizes below a piece, dW in parts, sums in parts; rows that are no expert's
@pytest.mark.parametrize("shift", [0, 1, 5])
@pytest.mark.parametrize("counts,extra,n,k,dtype", [
    ([3, 0, 2], 1, 40, 96, torch.bfloat16), ([200, 3, 31], 5, 264, 200, torch.bfloat16), ([128], 0, 1024, 4096, torch.bfloat16),
    ([200], 3, 515, 2051, torch.bfloat16), ([2000, 0, 2040], 9, 2048, 2056, torch.bfloat16), ([2040, 2000], 7, 2041, 4099, torch.bfloat16),
    ([3000, 1090], 0, 4096, 1000, torch.bfloat16), ([9001, 0], 2, 264, 72, torch.bfloat16), ([70, 9, 0, 300], 3, 5, 90, torch.bfloat16),
    ([3, 0, 2], 1, 7, 33, torch.float32), ([500, 300], 9, 193, 333, torch.float32), ([5003], 1, 66, 70, torch.float32),
    ([1500, 2600, 900], 3, 512, 1028, torch.float32), ([70, 9, 0, 300], 3, 3, 300, torch.float32)])
def test_products(counts, extra, n, k, dtype, shift):
    gen = torch.Generator("cuda").manual_seed(n + k)
    rows, experts = sum(counts) + extra, len(counts)
    x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(experts, n, k, generator=gen, device="cuda").to(dtype).requires_grad_()
    g = torch.randn(rows, n, generator=gen, device="cuda").to(dtype)
    ends = torch.tensor(counts, device="cuda").cumsum(0).int()
    y = ab.expert_mm(x, w, ends)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    # operands at another address may take another kernel: whole 16-byte pieces or not, the same sums in another order
    size = 2.0 ** -7 if dtype == torch.bfloat16 else 1e-4
    xi, wi, gi, ei = (_inside(t.detach(), s) for t, s in ((x, shift), (w, shift), (g, shift), (ends, 1)))
    for product, (name, a, b, want) in enumerate((("adambridge_expert_mm", xi, wi, y), ("adambridge_expert_mm_dx", gi, wi, dx),
                                                  ("adambridge_expert_mm_dw", gi, xi, dw))):
        work = _work("adambridge_expert_mm_work", product, CODES[dtype], rows, experts, n, k)
        out = _Result(want.shape, dtype, shift)
        _call(name, a, b, ei, out, CODES[dtype], rows, experts, n, k, work)
        out.check(want.detach(), None if shift == 0 else dict(rtol=size, atol=size * want.detach().float().std().item()))
        if work is not None:
            assert (work.whole[:GUARD] == -7).all() and (work.whole[GUARD + work.n:] == -7).all()


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 7), (70, 130), (3, 1025), (2100, 1999), (40, 4099), (7, 8192), (2050, 5003), (3, 16390), (2, 33000)])
def test_norms(rows, cols, dtype, w_dtype, shift):
    gen = torch.Generator("cuda").manual_seed(cols)
    x = torch.randn(rows, cols, generator=gen, device="cuda").to(dtype).requires_grad_()
    w, b = (torch.randn(cols, generator=gen, device="cuda").to(w_dtype).requires_grad_() for _ in range(2))
    g = torch.randn(rows, cols, generator=gen, device="cuda").to(dtype)
    y = ab.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), g)
    xi, gi, wi, bi = (_inside(t.detach(), shift) for t in (x, g, w, b))
    out, stats = _Result((rows, cols), dtype, shift), _Result((rows, 2), torch.float32, shift)
    _call("adambridge_layer_norm", xi, CODES[dtype], wi, bi, CODES[w_dtype], rows, cols, 1e-5, out, stats)
    out.check(y.detach())
    stats.check(stats.value)
    work = _work("adambridge_layer_norm_work", rows, cols, CODES[dtype])
    outs = [_Result(t.shape, t.dtype, shift) for t in grads]
    _call("adambridge_layer_norm_backward", gi, xi, CODES[dtype], wi, CODES[w_dtype], stats, rows, cols, *outs, work)
    for got, want in zip(outs, grads):
        got.check(want)
    assert (work.whole[:GUARD] == -7).all() and (work.whole[GUARD + work.n:] == -7).all()


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,experts,k,cols", [(1, 1, 1, 1), (7, 8, 2, 897), (64, 17, 5, 8), (65, 33, 17, 513), (300, 300, 8, 40), (4099, 16, 3, 1500)])
def test_routing_and_shuffles(tokens, experts, k, cols, dtype, shift):
    gen = torch.Generator("cuda").manual_seed(tokens + experts)
    logits = torch.randn(tokens, experts, generator=gen, device="cuda").to(dtype).requires_grad_()
    gw = torch.randn(tokens, k, generator=gen, device="cuda")
    code = CODES[dtype]
    for normalize in (1, 0):
        r = ab.route(logits, k, normalize=bool(normalize))
        dlogits, = torch.autograd.grad(r.weights, logits, gw)
        li, gi = _inside(logits.detach(), shift), _inside(gw, shift)
        outs = [_Result(t.shape, t.dtype, shift) for t in r]
        work = _work("adambridge_route_work", tokens, experts, k)
        _call("adambridge_route", li, code, tokens, experts, k, normalize, *outs, work)
        for got, want in zip(outs, r):
            got.check(want.detach())
        if work is not None:
            assert (work.whole[:GUARD] == -7).all() and (work.whole[GUARD + work.n:] == -7).all()
        grad = _Result(dlogits.shape, dtype, shift)
        _call("adambridge_route_backward", outs[0], outs[1], gi, li, code, tokens, experts, k, normalize, grad)
        grad.check(dlogits)
    x = torch.randn(tokens, cols, generator=gen, device="cuda").to(dtype)
    y = torch.randn(tokens * k, cols, generator=gen, device="cuda").to(dtype).requires_grad_()
    weights = r.weights.detach().clone().requires_grad_()
    out = ab.combine(y, r._replace(weights=weights))
    dy, dw = torch.autograd.grad(out, (y, weights), x)
    xi, yi, wi, pi = _inside(x, shift), _inside(y.detach(), shift), _inside(weights.detach(), shift), _inside(r.position, shift)
    rows = _Result((tokens * k, cols), dtype, shift)
    _call("adambridge_dispatch", xi, code, pi, tokens, k, cols, rows)
    rows.check(ab.dispatch(x, r))
    got = _Result((tokens, cols), dtype, shift)
    _call("adambridge_combine", yi, code, wi, pi, tokens, k, cols, got)
    got.check(out.detach())
    drows, dweights = _Result(dy.shape, dtype, shift), _Result(dw.shape, torch.float32, shift)
    _call("adambridge_combine_backward", xi, yi, code, wi, pi, tokens, k, cols, drows, dweights)
    drows.check(dy)
    dweights.check(dw)


# experts whose rows and weights are NaN beside others, in the tiled kernels (neighbours share their tiles' loads)
@pytest.mark.parametrize("counts,extra,n,k,dtype", [
    ([2000, 33, 2040], 9, 2048, 2056, torch.bfloat16), ([2040, 100, 1900], 7, 2041, 4099, torch.bfloat16), ([200, 60, 190], 5, 264, 2200, torch.bfloat16),
    ([4000, 300, 4001], 9, 136, 72, torch.bfloat16), ([1500, 70, 900], 5, 512, 1028, torch.float32), ([700, 9, 300], 3, 3, 300, torch.float32),
    ([700, 9, 300], 3, 90, 5, torch.bfloat16)])
def test_what_an_expert_holds_stays_with_it(counts, extra, n, k, dtype):
    gen = torch.Generator("cuda").manual_seed(n + k)
    rows = sum(counts) + extra
    x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype)
    w = torch.randn(3, n, k, generator=gen, device="cuda").to(dtype)
    g = torch.randn(rows, n, generator=gen, device="cuda").to(dtype)
    ends = torch.tensor(counts, device="cuda").cumsum(0).int()
    results = []
    for poisoned in (False, True):
        if poisoned:
            lo, hi = counts[0], counts[0] + counts[1]
            x[lo:hi], g[lo:hi], w[1] = torch.nan, torch.inf, torch.nan
            x[sum(counts):], g[sum(counts):] = torch.inf, torch.nan
        leaves = [t.clone().requires_grad_() for t in (x, w)]
        y = ab.expert_mm(*leaves, ends)
        results.append((y.detach(), *torch.autograd.grad(y, leaves, g)))
    clean, dirty = results
    others = torch.ones(rows, dtype=torch.bool, device="cuda")
    others[counts[0]:counts[0] + counts[1]] = False
    for i in range(2):
        assert torch.equal(clean[i][others], dirty[i][others]) and dirty[i][~others].isnan().all()
    assert torch.equal(clean[2][[0, 2]], dirty[2][[0, 2]]) and dirty[2][1].isnan().all()
