"""The expert layer's operators by the library's kernels (csrc/abh_route.hip, csrc/abh_experts.hip) against their
definitions in 64 bits."""

import pytest
import torch

import adambridge_amd as ab
from adambridge_amd import _hip, experts

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -23}   # twice the half ulp a rounding costs


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


# ----------------------------------------------------------------------- route

def _exact_route(logits, k, normalize):
    wide = logits.detach().double()
    # float64 keys that order as the definition does: NaN above +inf
    keys = torch.where(wide.isnan(), torch.finfo(torch.float64).max, wide.clamp(max=1e300))
    left, chosen = keys.clone(), []
    index = torch.arange(wide.shape[1], device="cuda").expand_as(left)
    taken = torch.zeros_like(left, dtype=torch.bool)
    for _ in range(k):
        best = left.masked_fill(taken, -torch.inf)
        top = best.amax(1, keepdim=True)
        at = torch.where((best == top) & ~taken, index, wide.shape[1]).amin(1)
        chosen.append(at)
        taken[torch.arange(len(at), device="cuda"), at] = True
    chosen = torch.stack(chosen, 1)
    hot = torch.zeros(wide.shape, dtype=torch.int64, device="cuda").scatter_(1, chosen, 1)
    ends = hot.sum(0).cumsum(0)
    position = (ends - hot.sum(0))[chosen] + torch.gather(hot.cumsum(0) - hot, 1, chosen)
    source = wide.clone().requires_grad_()
    weights = (torch.softmax(torch.gather(source, 1, chosen), 1) if normalize
               else torch.gather(torch.softmax(source, 1), 1, chosen))
    return chosen, ends, position, torch.argsort(position.reshape(-1)), weights, source


def _check_route(logits, k, normalize, seed=0):
    leaf = logits.detach().requires_grad_()
    r = ab.route(leaf, k, normalize=normalize)
    chosen, ends, position, order, weights, source = _exact_route(logits, k, normalize)
    assert all(t.dtype == torch.int32 for t in r[1:]) and r.weights.dtype == torch.float32
    for got, want in zip(r[1:], (chosen, ends, order, position)):
        assert torch.equal(got.long(), want)
    # exp's argument is off by 2^-24 of |x - max| log2(e), below 2^5.5 here; the sum's and the quotient's roundings
    assert ((r.weights.double() - weights).abs() <= weights * 2.0 ** -17 + 1e-38).all()
    g = torch.randn(weights.shape, generator=_gen(seed + 1), device="cuda")
    grad, = torch.autograd.grad(r.weights, leaf, g)
    want, = torch.autograd.grad(weights, source, g.double())
    assert grad.dtype == logits.dtype
    p = torch.softmax(logits.double(), 1) if not normalize else torch.zeros(logits.shape, dtype=torch.float64, device="cuda").scatter_(
        1, chosen, weights.detach())
    # dlogit = p (g - sum p g): each factor off by 2^-17 of its size
    size = p * (g.abs().amax(1, keepdim=True) * 2.0)
    assert ((grad.double() - want).abs() <= want.abs() * UNIT[logits.dtype] + size * 2.0 ** -15 + 1e-38).all()
    with torch.no_grad():
        again = ab.route(logits, k, normalize=normalize)
    assert all(torch.equal(a, b) for a, b in zip(again, r))


# one token and one expert; the ends of a block of 64 tokens and of every number of lanes and logits a lane; more choices
# than a short group has lanes; several blocks, the last not whole
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,n,k", [(1, 1, 1), (1, 64, 4), (3, 2, 2), (63, 16, 16), (64, 17, 2), (65, 33, 17), (130, 65, 8),
                                        (257, 128, 8), (1000, 256, 6), (67, 257, 64), (90, 1024, 33), (4161, 8, 2)])
def test_route_matches_the_definition(tokens, n, k, dtype, normalize):
    logits = (torch.randn(tokens, n, generator=_gen(tokens + n), device="cuda") * 2.0).to(dtype)
    _check_route(logits, k, normalize)


def test_route_takes_the_lower_index_of_equal_logits():
    logits = torch.randint(0, 3, (200, 40), generator=_gen(3), device="cuda").float()
    logits[::7] = 0.0
    logits[1::7] *= -0.0   # +0 and -0 are equal
    _check_route(logits, 6, True)
    _check_route(logits.bfloat16(), 6, False)


@pytest.mark.parametrize("normalize", [True, False])
def test_route_of_masked_infinite_and_nan_logits(normalize):
    logits = torch.randn(70, 20, generator=_gen(4), device="cuda")
    logits[:, 5:] = -torch.inf                                # fewer than are chosen are left in some rows
    logits[1, :] = -torch.inf
    logits[2, 1:] = -torch.inf
    logits[3] = torch.finfo(torch.float32).min
    logits[4, 7], logits[5, 3] = torch.nan, torch.inf
    leaf = logits.clone().requires_grad_()
    r = ab.route(leaf, 6, normalize=normalize)
    cpu_leaf = logits.cpu().requires_grad_()
    want = ab.route(cpu_leaf, 6, normalize=normalize)
    for got, w in zip(r[1:], want[1:]):
        assert torch.equal(got.cpu(), w)
    assert torch.allclose(r.weights.cpu(), want.weights, rtol=1e-5, atol=1e-30, equal_nan=True)
    assert torch.equal(r.experts[1].cpu(), torch.arange(6, dtype=torch.int32)) and not r.weights[1].any()
    assert r.experts[4, 0] == 7 and r.weights[4].isnan().all() and r.weights[5].isnan().any()
    keep = [i for i in range(70) if i not in (4, 5)]
    r = ab.route(leaf[keep], 6, normalize=normalize)
    want = ab.route(cpu_leaf[keep], 6, normalize=normalize)
    g = torch.randn(68, 6, generator=_gen(5), device="cuda")
    grad, = torch.autograd.grad(r.weights, leaf, g)
    want_grad, = torch.autograd.grad(want.weights, cpu_leaf, g.cpu())
    assert torch.isfinite(grad[keep]).all() and not grad[1].any()
    rows = [i for i in keep if i != 1]
    assert torch.allclose(grad[rows].cpu(), want_grad[rows], rtol=1e-4, atol=1e-6)


def test_route_gradient_against_differences():
    logits = torch.randn(9, 12, generator=_gen(6), device="cuda") * 3.0
    g, d = torch.randn(9, 3, generator=_gen(7), device="cuda"), torch.randn(9, 12, generator=_gen(8), device="cuda")
    for normalize in (True, False):
        leaf = logits.clone().requires_grad_()
        grad, = torch.autograd.grad(ab.route(leaf, 3, normalize=normalize).weights, leaf, g)
        h = 2.0 ** -9   # no two logits of a row are near enough to change places
        up, down = (ab.route(logits + s * h * d, 3, normalize=normalize).weights.double() for s in (1, -1))
        want = ((up - down) * g.double()).sum() / (2 * h)
        assert abs(want - (grad.double() * d.double()).sum()) <= 27 * 2.0 ** -22 / h + 27 * 8 * h ** 2


# -------------------------------------------------------- dispatch and combine

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,n,k,hidden", [(1, 1, 1, 1), (7, 8, 2, 897), (5, 4, 4, 8), (130, 16, 3, 513), (66, 64, 8, 2048), (3, 9, 1, 4099)])
def test_dispatch_and_combine_match_the_definition(tokens, n, k, hidden, dtype):
    gen = _gen(tokens * hidden)
    r = ab.route(torch.randn(tokens, n, generator=gen, device="cuda"), k)
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype).requires_grad_()
    rows = ab.dispatch(x, r)
    token = r.order.long() // k
    assert torch.equal(rows, x[token])
    g = torch.randn(tokens * k, hidden, generator=gen, device="cuda").to(dtype)
    dx, = torch.autograd.grad(rows, x, g)
    picked = g.double()[r.position.long()]
    want = picked.sum(1)
    # k terms summed in FP32, one rounding
    assert ((dx.double() - want).abs() <= want.abs() * UNIT[dtype] + picked.abs().sum(1) * k * 2.0 ** -23).all()

    y = torch.randn(tokens * k, hidden, generator=gen, device="cuda").to(dtype).requires_grad_()
    weights = r.weights.clone().requires_grad_()
    out = ab.combine(y, r._replace(weights=weights))
    terms = y.detach().double()[r.position.long()] * r.weights.double()[:, :, None]
    want = terms.sum(1)
    assert ((out.double() - want).abs() <= want.abs() * UNIT[dtype] + terms.abs().sum(1) * k * 2.0 ** -23).all()
    g = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype)
    dy, dw = torch.autograd.grad(out, (y, weights), g)
    want = r.weights.double().reshape(-1)[r.order.long()][:, None] * g.double()[token]
    assert ((dy.double() - want).abs() <= want.abs() * UNIT[dtype]).all()
    products = y.detach().double()[r.position.long()] * g.double()[:, None, :]
    # a lane's hidden / 64 terms and a tree: below hidden / 64 + 8 roundings of the partial sums
    assert ((dw.double() - products.sum(2)).abs() <= products.abs().sum(2) * (hidden / 64 + 16) * 2.0 ** -23).all()
    # each gradient alone
    for leaf, grad in ((y, dy), (weights, dw)):
        alone = [t.detach().requires_grad_(t is leaf) for t in (y, weights)]
        got, = torch.autograd.grad(ab.combine(alone[0], r._replace(weights=alone[1])), [t for t in alone if t.requires_grad], g)
        assert torch.equal(got, grad)


def test_rows_of_no_routing_are_left_out():
    """A position outside the rows counts as zeros, and nothing is written for it."""
    r = ab.route(torch.randn(4, 6, generator=_gen(1), device="cuda"), 2)
    position = r.position.clone()
    position[1, 1], position[3, 0] = 8, -1
    bad = r._replace(position=position)
    y = torch.randn(8, 40, generator=_gen(2), device="cuda")
    keep = torch.ones_like(r.weights)
    keep[1, 1] = keep[3, 0] = 0.0
    assert torch.equal(ab.combine(y, bad), ab.combine(y, r._replace(weights=r.weights * keep)))
    dw = _hip.load().combine_backward(torch.ones(4, 40, device="cuda"), y, r.weights, position, (True, True))[1]
    assert dw[1, 1] == 0.0 and dw[3, 0] == 0.0


# ------------------------------------------------------------------- expert_mm

def _ends(counts, device="cuda"):
    return torch.tensor(counts, device=device).cumsum(0).int()


def _check_mm(counts, extra, n, k, dtype, seed=0, ends=None):
    gen = _gen(seed)
    rows, e = sum(counts) + extra, len(counts)
    x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(e, n, k, generator=gen, device="cuda").to(dtype).requires_grad_()
    g = torch.randn(rows, n, generator=gen, device="cuda").to(dtype)
    ends = _ends(counts) if ends is None else ends
    out = ab.expert_mm(x, w, ends)
    dx, dw = torch.autograd.grad(out, (x, w), g)
    with torch.no_grad():
        assert torch.equal(ab.expert_mm(x, w, ends), out)
    assert out.dtype == dx.dtype == dw.dtype == dtype
    lo = 0
    unit = UNIT[dtype]

    def near(got, a, b):
        """got = a b: sums of len terms in FP32, whatever their order, and one rounding."""
        want, size = a @ b, a.abs() @ b.abs()
        assert ((got.double() - want).abs() <= want.abs() * unit + size * max(1, a.shape[1]) * 2.0 ** -23).all()

    for i, count in enumerate(counts):
        hi = lo + count
        xe, we, ge = x.detach()[lo:hi].double(), w.detach()[i].double(), g[lo:hi].double()
        near(out[lo:hi], xe, we.t())
        near(dx[lo:hi], ge, we)
        near(dw[i], ge.t(), xe)
        lo = hi
    assert not out[lo:].any() and not dx[lo:].any()
    return out, dx, dw


# one row and one value; odd sizes on both sides of every tile and step; experts without rows first, between and last;
# rows that are no expert's; one expert with all rows; more experts than a wavefront has lanes
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,extra,n,k", [
    ([1], 0, 1, 1), ([3, 0, 2], 0, 7, 5), ([0, 129, 1, 0], 3, 130, 33), ([0, 0, 300], 0, 64, 257), ([128, 127, 129], 0, 127, 129),
    ([5, 1, 1, 1], 0, 256, 512), ([1] * 8, 0, 96, 2048), ([2, 0] * 70 + [9], 5, 40, 48), ([0, 0], 4, 24, 40), ([700], 0, 264, 200),
    ([257, 0, 31, 513], 0, 520, 320), ([16, 17, 1, 30], 2, 192, 1000)])
def test_expert_mm_matches_the_definition(counts, extra, n, k, dtype):
    _check_mm(counts, extra, n, k, dtype, seed=n + k)


# what the smaller sizes do not reach: whole rounds of large tiles and a rest that is cut along its sum (of y and of dx), a
# last tile of few rows, a dW of few tiles in parts of its rows; each with and without rows of whole 16-byte pieces
@pytest.mark.parametrize("counts,extra,n,k,dtype", [
    ([2000, 0, 2040], 0, 4096, 2048, torch.bfloat16), ([2040, 2000], 7, 2041, 4099, torch.bfloat16),
    ([3000, 1090], 0, 4099, 2043, torch.bfloat16), ([70, 300, 2500, 90, 5300], 0, 2048, 4224, torch.bfloat16),
    ([9001, 0], 0, 264, 72, torch.bfloat16), ([4000, 3001], 9, 130, 67, torch.bfloat16), ([5003], 0, 66, 70, torch.float32),
    ([1500, 2600, 900], 0, 512, 1028, torch.float32), ([64, 3, 0, 61] * 40, 0, 1024, 520, torch.bfloat16)])
def test_expert_mm_of_many_rows_matches_the_definition(counts, extra, n, k, dtype):
    _check_mm(counts, extra, n, k, dtype, seed=n + k)


# few tiles, whose sums are cut into parts (of y over k, of dx over n), the last one short; rows that are no expert's
@pytest.mark.parametrize("counts,extra,n,k", [([128], 0, 1024, 4096), ([100, 0, 90], 5, 1000, 2056), ([200], 3, 515, 2051),
                                              ([40], 0, 1024, 8200), ([150], 0, 4096, 520), ([60, 70], 1, 2049, 129)])
def test_expert_mm_of_few_tiles_matches_the_definition(counts, extra, n, k):
    _check_mm(counts, extra, n, k, torch.bfloat16, seed=n + k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_rows_at_all(dtype):
    x = torch.randn(0, 24, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(3, 16, 24, device="cuda").to(dtype).requires_grad_()
    out = ab.expert_mm(x, w, _ends([0, 0, 0]))
    assert out.shape == (0, 16)
    dx, dw = torch.autograd.grad(out, (x, w), torch.zeros_like(out))
    assert dx.shape == (0, 24) and dw.shape == w.shape and not dw.any()


@pytest.mark.parametrize("n,k", [(64, 128), (61, 35)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan_stay_with_their_expert(n, k, dtype):
    counts = [40, 3, 0, 65]
    clean = _check_mm(counts, 6, n, k, dtype)
    gen = _gen(0)
    x = torch.randn(114, k, generator=gen, device="cuda").to(dtype)
    w = torch.randn(4, n, k, generator=gen, device="cuda").to(dtype)
    g = torch.randn(114, n, generator=gen, device="cuda").to(dtype)
    x[41], g[42], w[1] = torch.nan, torch.inf, torch.nan    # all of the second expert's
    w[2] = torch.nan                                          # an expert without rows
    x[108:], g[108:] = torch.nan, torch.inf                   # rows that are no expert's
    x.requires_grad_(), w.requires_grad_()
    out = ab.expert_mm(x, w, _ends(counts))
    dx, dw = torch.autograd.grad(out, (x, w), g)
    rows = [i for i in range(114) if not 40 <= i < 43]
    assert torch.equal(out[rows], clean[0][rows]) and torch.equal(dx[rows], clean[1][rows])
    assert torch.equal(dw[[0, 2, 3]], clean[2][[0, 2, 3]]) and not dw[2].any()
    assert out[40:43].isnan().all() and dw[1].isnan().all()


def test_ends_beyond_the_rows_are_the_rows_end():
    x, w = torch.randn(20, 16, device="cuda"), torch.randn(3, 8, 16, device="cuda")
    assert torch.equal(ab.expert_mm(x, w, torch.tensor([5, 90, 100], device="cuda", dtype=torch.int32)),
                       ab.expert_mm(x, w, torch.tensor([5, 20, 20], device="cuda", dtype=torch.int32)))


def test_strided_operands_autocast_and_the_second_derivative():
    gen = _gen(9)
    x = torch.randn(30, 48, generator=gen, device="cuda")
    w = torch.randn(2, 48, 24, generator=gen, device="cuda")
    ends = _ends([13, 17])
    want = ab.expert_mm(x, w.transpose(1, 2).contiguous(), ends)
    leaf = w.clone().requires_grad_()
    out = ab.expert_mm(x.t().contiguous().t(), leaf.transpose(1, 2), ends)
    assert torch.equal(out, want)
    dw, = torch.autograd.grad(out, leaf, torch.ones(1, 1, device="cuda").expand(30, 24))
    assert torch.allclose(dw[0], x[:13].sum(0)[:, None].expand(48, 24), rtol=1e-5, atol=1e-4)
    wt = w.transpose(1, 2).contiguous().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = ab.expert_mm(x, wt, ends)
    assert out.dtype == torch.bfloat16 and torch.equal(out, ab.expert_mm(x.bfloat16(), wt.detach().bfloat16(), ends))
    assert torch.autograd.grad(out.float().sum(), wt)[0].dtype == torch.float32
    xl = x.clone().requires_grad_()
    dx, = torch.autograd.grad(ab.expert_mm(xl, wt, ends).square().sum(), xl, create_graph=True)
    got, = torch.autograd.grad(dx.sum(), wt)
    xc, wc = x.cpu().requires_grad_(), wt.detach().cpu().requires_grad_()
    dx, = torch.autograd.grad(ab.expert_mm(xc, wc, ends.cpu()).square().sum(), xc, create_graph=True)
    assert torch.allclose(got.cpu(), torch.autograd.grad(dx.sum(), wc)[0], rtol=1e-3, atol=1e-2)


def test_gradient_against_differences():
    """expert_mm is linear in each operand: differences are exact but for rounding."""
    gen = _gen(11)
    ends = _ends([7, 0, 22])
    leaves = [torch.randn(29, 50, generator=gen, device="cuda").requires_grad_(),
              torch.randn(3, 33, 50, generator=gen, device="cuda").requires_grad_()]
    g = torch.randn(29, 33, generator=gen, device="cuda")
    grads = torch.autograd.grad(ab.expert_mm(*leaves, ends), leaves, g)
    with torch.no_grad():
        for i in range(2):
            d = torch.randn(leaves[i].shape, generator=gen, device="cuda")
            up, down = (ab.expert_mm(*[t + s * d if j == i else t for j, t in enumerate(leaves)], ends).double() for s in (1, -1))
            want = ((up - down) * g.double()).sum() / 2
            # 957 outputs below 64, rounded to 2^-18 of them at 50 terms each, times g
            assert abs(want - (grads[i].double() * d.double()).sum()) <= 957 ** 0.5 * 64 * 50 * 2.0 ** -23


def test_the_kernels_run_and_refuse_wrong_operands(monkeypatch):
    k = _hip.load()
    x, w = torch.randn(6, 16, device="cuda"), torch.randn(2, 8, 16, device="cuda")
    ends = _ends([2, 4])
    with pytest.raises(ValueError, match="x must be contiguous"):
        k.expert_mm(x.t(), w, ends)
    with pytest.raises(ValueError, match="weight must be contiguous"):
        k.expert_mm(x, w.bfloat16(), ends)
    with pytest.raises(ValueError, match="ends must be contiguous"):
        k.expert_mm(x, w, ends.long())
    with pytest.raises(ValueError, match="gout must be contiguous"):
        k.expert_mm_backward(x, x, w, ends, (True, True))
    with pytest.raises(ValueError, match="position must be contiguous"):
        k.dispatch(x, torch.zeros(5, 2, dtype=torch.int32, device="cuda"))
    for name in ("_torch_route", "_torch_dispatch", "_torch_gather_sum", "_torch_rows"):
        monkeypatch.setattr(experts, name, None)   # ordinary calls do not come here
    r = ab.route(torch.randn(6, 2, device="cuda"), 1)
    ab.combine(ab.expert_mm(ab.dispatch(x, r), w, r.ends), r)


# --------------------------------------------------------------- the whole block

def _block(x, gate, up, down, norm, k=2):
    h = ab.layer_norm(x, *norm)
    r = ab.route(h @ gate.t(), k)
    rows = torch.nn.functional.gelu(ab.expert_mm(ab.dispatch(h, r), up, r.ends))
    return x + ab.combine(ab.expert_mm(rows, down, r.ends), r)


def _block_case(dtype=torch.bfloat16, tokens=100, hidden=128, inter=192, n=6):
    gen = _gen(21)
    shapes = [(n, hidden), (n, inter, hidden), (n, hidden, inter)]
    params = [(torch.randn(*s, generator=gen, device="cuda") * 0.1).to(dtype).requires_grad_() for s in shapes]
    norm = [torch.ones(hidden, device="cuda", dtype=dtype).requires_grad_(), torch.zeros(hidden, device="cuda", dtype=dtype).requires_grad_()]
    return torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype).requires_grad_(), params, norm


def test_a_block_on_another_stream_and_twice():
    """The same bits again, on whatever stream is current, the gradients' included."""
    x, params, norm = _block_case()
    leaves = [x, *params, *norm]

    def once():
        out = _block(x, *params, norm)
        return (out, *torch.autograd.grad(out.float().square().sum(), leaves))

    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_block_captured_in_a_graph():
    x, params, norm = _block_case()
    leaves = [x, *params, *norm]

    def once():
        out = _block(x, *params, norm)
        return (out, *torch.autograd.grad(out, leaves, seed))

    seed = torch.randn(x.shape, generator=_gen(3), device="cuda").to(x.dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=_gen(30 + i), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = once()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), i
