"""How near the expert products come to their definition in 64 bits, result by result in norm: sums that were kept in
fewer bits than 32, or in one long chain where they are said to be in short ones, are further away."""

import pytest
import torch

import adambridge_amd as ab

CHAIN = 256   # terms that an FP32 product adds up one after the other


def _ends(counts):
    return torch.tensor(counts, device="cuda").cumsum(0).int()


def fp32_bound(terms):
    """Norm of the error over the result's, for normal operands.  A chain of L additions of size-growing sums loses
    at most 2^-24 of each partial sum, independently: 2^-24 sqrt(L / 2) of the result (its last sum) as a root mean
    square.  Chains of CHAIN terms, whose results are added in chains again, or in parts: no more chains than there are."""
    return 2.0 ** -24 * ((min(terms, CHAIN) + -(-terms // CHAIN)) / 2 + 1) ** 0.5


def bf16_bound(terms):
    """Norm of the difference to the rounded definition over the result's.  A result changes its rounding if it is
    within an FP32 sum's error of a tie, of which there is one each ulp, 2^-8 of the value or more: a part
    2 2^-24 sqrt(terms / 2) / 2^-8 of the results, by an ulp."""
    return 2.0 ** -7.5 * (2.0 ** -15 * (terms / 2 + 1) ** 0.5) ** 0.5


def _near(got, a, b):
    if not a.numel() or not b.numel() or got.numel() < 1000:   # few results: no norm to speak of
        return
    want, terms = a @ b, a.shape[1]
    if got.dtype == torch.bfloat16:
        error, bound = got.double() - want.bfloat16().double(), bf16_bound(terms)
    else:
        error, bound = got.double() - want, fp32_bound(terms)
    assert error.norm() <= bound * want.norm(), (terms, (error.norm() / want.norm()).item(), bound)


def _check(counts, n, k, dtype, extra=0):
    gen = torch.Generator("cuda").manual_seed(n + k)
    rows = sum(counts) + extra
    x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(len(counts), n, k, generator=gen, device="cuda").to(dtype).requires_grad_()
    g = torch.randn(rows, n, generator=gen, device="cuda").to(dtype)
    out = ab.expert_mm(x, w, _ends(counts))
    dx, dw = torch.autograd.grad(out, (x, w), g)
    lo = 0
    for e, count in enumerate(counts):
        xe, we, ge = (t.detach().double() for t in (x[lo:lo + count], w[e], g[lo:lo + count]))
        _near(out[lo:lo + count], xe, we.t())
        _near(dx[lo:lo + count], ge, we)
        _near(dw[e], ge.t().contiguous(), xe)
        lo += count


# streamed, whole tiles, tiles cut along their sums, rests of a round, weights' gradients in parts, odd sizes of each
@pytest.mark.gpu
@pytest.mark.parametrize("counts,n,k,dtype", [
    ([9, 7], 1024, 8200, torch.float32), ([60, 64, 2], 2048, 4096, torch.float32), ([5003], 66, 70, torch.float32),
    ([1500, 2600, 900], 512, 1028, torch.float32), ([300, 200], 4099, 5003, torch.float32), ([4000, 9000], 512, 520, torch.float32),
    ([2000, 0, 2040], 4096, 2048, torch.bfloat16), ([2040, 2000], 2041, 4099, torch.bfloat16),
    ([70, 300, 2500, 90, 5300], 2048, 4224, torch.bfloat16), ([9001, 0], 264, 72, torch.bfloat16), ([4000, 3001], 130, 67, torch.bfloat16),
    ([128], 1024, 4096, torch.bfloat16), ([200], 515, 2051, torch.bfloat16), ([40], 1024, 8200, torch.bfloat16),
    ([150], 4096, 520, torch.bfloat16), ([3, 9, 0, 1], 1536, 4096, torch.bfloat16)])
def test_products_in_norm(counts, n, k, dtype):
    _check(counts, n, k, dtype)


# sizes below a 16-byte piece over many rows
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts,n,k", [([60000, 5000], 3, 1000), ([70001], 1000, 3), ([40000, 0, 25000], 2, 515)])
def test_weights_gradients_of_narrow_layers_in_norm(counts, n, k, dtype):
    _check(counts, n, k, dtype)


def test_the_bounds_tell_narrower_sums_apart():
    """Sums kept in fewer bits, planted in the oracle on the CPU, are beyond the bounds."""
    gen = torch.Generator().manual_seed(0)
    for terms in (1028, 2048, 4096):
        a, b = (torch.randn(*s, generator=gen) for s in ((64, terms), (terms, 64)))
        want = a.double() @ b.double()
        cut = lambda t, bits: (t.view(torch.int32) & -(1 << (23 - bits))).view(torch.float32)
        for bits in (10, 12, 16):
            error = cut(a, bits).double() @ cut(b, bits).double() - want
            assert error.norm() > fp32_bound(terms) * want.norm()
        a, b = a.bfloat16(), b.bfloat16()
        want = a.double() @ b.double()
        parts = sum((a[:, i::4].float() @ b[i::4].float()).bfloat16() for i in range(4))   # each part rounded
        error = parts.double() - want.bfloat16().double()
        assert error.norm() > bf16_bound(terms) * want.norm()
    a, b = (torch.randn(*s, generator=gen) for s in ((32, 65536), (65536, 32)))
    chain = torch.zeros(32, 32)
    for i in range(65536):   # one chain of 65536
        chain += a[:, i:i + 1] * b[i:i + 1]
    want = a.double() @ b.double()
    assert (chain.double() - want).norm() > fp32_bound(65536) * want.norm()
