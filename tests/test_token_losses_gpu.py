"""token_losses' kernels against the definition in 64 bits: sizes about the tiles and the pieces of the vocabulary, rows that are not
scored, targets outside the vocabulary."""

import pytest
import torch

import adambridge_amd as ab

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
U = 2.0 ** -24   # FP32's largest relative rounding


def _definition(h, w, t, gout, ignore):
    """Losses and gradients in 64 bits, and bounds of the kernels' errors, in slices of rows."""
    eps = torch.finfo(h.dtype).eps / 2
    h, w = h.double(), w.double()
    rows, size = h.shape
    vocab = w.shape[0]
    losses, loss_bounds, dhs, dh_bounds = [], [], [], []
    dw, dw_bound = torch.zeros_like(w), torch.zeros_like(w)
    for lo in range(0, rows, 8192):
        scored = t[lo:lo + 8192] != ignore
        a = torch.where(scored[:, None], h[lo:lo + 8192], 0.0)
        hot = (t[lo:lo + 8192, None] == torch.arange(vocab, device="cuda")).double()
        x = a @ w.t()
        losses.append(torch.where(scored, torch.logsumexp(x, 1) - (x * hot).sum(1), 0.0))
        # a logit: `size` exact products summed in FP32; the sum of exponentials: a lane's, then tiles' in turn, fewer than 1024 roundings
        # one after the other, an exponential's exponent, below 2^7, rounded twice
        logit = (a.abs() @ w.abs().t()).amax(1) * (size + 1) * U
        wrong = 2 * logit + (1024 + 2 * 128) * U
        loss_bounds.append(wrong + 4 * U * losses[-1].abs() + 2 * U * x.abs().amax(1))
        p = torch.softmax(x, 1)
        g = torch.where(scored, gout[lo:lo + 8192].double(), 0.0)[:, None]
        dhs.append((p - hot) * g @ w)
        # G: the exponential's error and the sum's, its rounding to the type; then its products' sums
        large = (p + hot) * g.abs()
        each = (2 * wrong[:, None] + eps + 8 * U) * large
        dh_bounds.append(each @ w.abs() + large @ w.abs() * (vocab + 8) * U)
        dw += ((p - hot) * g).t() @ a
        dw_bound += each.t() @ a.abs() + large.t() @ a.abs() * (rows + 8) * U
    dh = torch.cat(dhs)
    return (torch.cat(losses), torch.cat(loss_bounds), dh, torch.cat(dh_bounds) + dh.abs() * eps, dw, dw_bound + dw.abs() * eps)


def _inputs(rows, vocab, size, dtype, gen, ignored=0.2):
    h = torch.randn(rows, size, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(vocab, size, generator=gen, device="cuda") * size ** -0.5 * 2).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    t[torch.rand(rows, generator=gen, device="cuda") < ignored] = -100
    return h, w, t, torch.rand(rows, generator=gen, device="cuda") + 0.25


def _check(h, w, t, gout, ignore=-100):
    want, loss_bound, dh, dh_bound, dw, dw_bound = _definition(h, w, t, gout, ignore)
    h, w = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ab.token_losses(h, w, t, ignore)
    assert loss.dtype == FP32 and loss.shape == t.shape
    assert ((loss.detach().double() - want).abs() <= loss_bound).all() and not loss[t == ignore].any()
    got = torch.autograd.grad(loss, (h, w), gout)
    assert ((got[0].double() - dh).abs() <= dh_bound).all() and not got[0][t == ignore].any()
    assert ((got[1].double() - dw).abs() <= dw_bound).all()
    with torch.no_grad():
        assert torch.equal(ab.token_losses(h, w, t, ignore), loss)
    for i, leaf in enumerate((h, w)):   # one of them alone, and again
        alone, = torch.autograd.grad(ab.token_losses(h, w, t, ignore), leaf, gout)
        assert torch.equal(alone, got[i])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,vocab,size", [
    (1, 1, 8), (1, 5003, 64), (3, 7, 9), (16, 64, 33), (17, 65, 264), (63, 1000, 100), (64, 17, 1030), (65, 1, 8), (65, 3, 16), (66, 9, 40),
    (257, 255, 264), (300, 257, 100), (600, 1000, 333), (1025, 5003, 72), (513, 30011, 24), (2100, 700, 1029), (130, 20000, 520)])
def test_losses_and_gradients(rows, vocab, size, dtype):
    gen = torch.Generator("cuda").manual_seed(rows + vocab + size)
    _check(*_inputs(rows, vocab, size, dtype, gen))


@pytest.mark.parametrize("dtype,size", [(FP32, 4), (FP32, 5), (BF16, 8), (BF16, 11)])
def test_the_shortest_rows(dtype, size):
    gen = torch.Generator("cuda").manual_seed(size)
    for rows in (5, 70):
        _check(*_inputs(rows, 50, size, dtype, gen))


@pytest.mark.parametrize("dtype,rows,vocab", [(BF16, 70000, 9001), (FP32, 66000, 4500)])
def test_pieces_of_the_vocabulary(dtype, rows, vocab):
    """More rows and words than one piece's gradient holds."""
    gen = torch.Generator("cuda").manual_seed(rows)
    _check(*_inputs(rows, vocab, 8, dtype, gen))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows", [9, 300])
def test_rows_that_are_not_scored(rows, dtype):
    """Whatever they hold reaches nothing; none scored gives zeros; targets are never read for them."""
    gen = torch.Generator("cuda").manual_seed(rows)
    h, w, t, gout = _inputs(rows, 500, 40, dtype, gen, 0.5)
    t[3] = 7
    results = []
    for poison in (0.0, torch.nan, torch.inf):
        here = torch.where((t == -100)[:, None], poison, h).to(dtype).requires_grad_()
        leaf = w.clone().requires_grad_()
        loss = ab.token_losses(here, leaf, t)
        g = torch.where(t == -100, poison, gout)
        results.append((loss.detach(), *torch.autograd.grad(loss, (here, leaf), g)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    here, leaf = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ab.token_losses(here, leaf, torch.full_like(t, 5), 5)
    assert not loss.any() and all(not g.any() for g in torch.autograd.grad(loss.sum(), (here, leaf)))
    _check(h, w, torch.where(t == -100, 499, t), gout, 7)


@pytest.mark.parametrize("rows", [9, 300])
def test_targets_outside_the_vocabulary(rows):
    gen = torch.Generator("cuda").manual_seed(rows)
    h, w, t, gout = _inputs(rows, 500, 40, FP32, gen)
    t[2], t[3], t[5] = 500, -1, 1 << 40
    here, leaf = h.requires_grad_(), w.requires_grad_()
    loss = ab.token_losses(here, leaf, t)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[2, 3, 5]] = True
    assert torch.equal(loss.isnan(), bad)
    dh, dw = torch.autograd.grad(loss, (here, leaf), gout)
    assert torch.equal(dh.isnan().all(1), bad) and torch.equal(dh.isnan().any(1), bad) and dw.isnan().all()


def test_infinite_logits():
    """A word that no row can reach (-inf); a row whose logits are all -inf, or hold a NaN or +inf, has no loss."""
    for rows in (12, 200):
        gen = torch.Generator("cuda").manual_seed(rows)
        h, w, t, _ = _inputs(rows, 300, 16, FP32, gen, 0.0)
        h = h.abs()
        w[17] = -torch.inf
        t[t == 17] = 18
        got, want = ab.token_losses(h, w, t), ab.token_losses(h, torch.cat((w[:17], w[18:])), torch.where(t > 17, t - 1, t))
        assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
        w[:] = -torch.inf
        assert ab.token_losses(h, w, t).isnan().all()
        w[:] = 1.0
        w[250] = torch.inf
        assert ab.token_losses(h, w, t).isnan().all()


def test_shapes_types_and_orders():
    gen = torch.Generator("cuda").manual_seed(3)
    h, w, t, gout = _inputs(210, 300, 48, BF16, gen)
    want = ab.token_losses(h, w, t)
    assert torch.equal(ab.token_losses(h.view(2, 3, 35, 48), w, t.view(2, 3, 35)), want.view(2, 3, 35))
    assert torch.equal(ab.token_losses(h, w, t.int()), want)
    assert torch.equal(ab.token_losses(h.t().contiguous().t(), w.t().contiguous().t(), torch.stack((t, t), 1)[:, 0]), want)
    assert torch.equal(ab.token_losses(h[0], w, t[0]), ab.token_losses(h[:1], w, t[:1])[0])
    assert ab.token_losses(h[:0], w, t[:0]).shape == (0,)
    wide = torch.zeros(300, 56, dtype=BF16, device="cuda")
    wide[:, 3:51] = w   # rows that are not at 16-byte boundaries
    assert torch.allclose(ab.token_losses(h, wide[:, 3:51], t), want)
    buffer = torch.zeros(300 * 48 + 1, dtype=BF16, device="cuda")
    buffer[1:] = w.reshape(-1)
    assert torch.allclose(ab.token_losses(h, buffer[1:].view(300, 48), t), want, rtol=1e-5, atol=1e-5)
    leaf, other = h.clone().requires_grad_(), h.clone().requires_grad_()
    summed, = torch.autograd.grad(ab.token_losses(leaf, w, t).sum(), leaf)   # a gradient that is one value in memory
    assert torch.equal(summed, torch.autograd.grad(ab.token_losses(other, w, t), other, torch.ones_like(gout))[0])
    tiny = torch.randn(9, 3, device="cuda"), torch.randn(20, 3, device="cuda"), torch.arange(9, device="cuda")
    assert torch.allclose(ab.token_losses(*tiny), torch.nn.functional.cross_entropy(tiny[0] @ tiny[1].t(), tiny[2], reduction="none"))
    with torch.autocast("cuda", dtype=BF16):
        assert torch.equal(ab.token_losses(h.float(), w.float(), t), want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,vocab,size,ignored", [
    (51, 74, 7540, 0.2), (1, 20, 8203, 0.0), (16, 1100, 2056, 0.2), (21, 1247, 2051, 0.2), (64, 37, 1030, 0.0), (1029, 342, 2053, 0.5),
    (3001, 185, 130, 0.2), (5000, 259, 1024, 0.9), (2049, 3, 1544, 0.97), (130, 5000, 1536, 0.2)])
def test_sums_of_few_tiles(rows, vocab, size, ignored, dtype):
    """Few tiles of long sums: the logits', dW's and dh's are cut along their terms, which may be fewer than the parts."""
    gen = torch.Generator("cuda").manual_seed(rows + vocab + size)
    _check(*_inputs(rows, vocab, size, dtype, gen, ignored))


@pytest.mark.parametrize("rows,vocab,size", [(2300, 4099, 2056), (4203, 4197, 2552), (4096, 4352, 2304)])
def test_sums_of_many_tiles(rows, vocab, size):
    """Many tiles of long sums, whose last step may be a part of one."""
    gen = torch.Generator("cuda").manual_seed(rows + vocab + size)
    _check(*_inputs(rows, vocab, size, BF16, gen))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_targets_and_logits_of_few_tiles(dtype):
    """Infinities, NaN and targets outside the vocabulary where the logits come in parts, as where they do not."""
    gen = torch.Generator("cuda").manual_seed(5)
    h, w, t, gout = _inputs(40, 70, 2048, dtype, gen, 0.0)
    t[0], t[1] = 70, -3
    h[2] = torch.nan
    w[:, 0] = 1.0
    h[3], h[4] = 0.0, 0.0
    h[3, 0], h[4, 0] = torch.inf, -torch.inf   # every logit inf, and -inf
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = ab.token_losses(h, w, t)
    dh, dw = torch.autograd.grad(loss, (h, w), gout)
    assert loss[:5].isnan().all() and dh[:5].isnan().all() and dw.isnan().all()
    rest = slice(5, None)
    want, bound, dh_want, dh_bound, _, _ = _definition(h.detach()[rest], w.detach(), t[rest], gout[rest], -100)
    assert ((loss.detach()[rest].double() - want).abs() <= bound).all()
    assert ((dh[rest].double() - dh_want).abs() <= dh_bound).all()
