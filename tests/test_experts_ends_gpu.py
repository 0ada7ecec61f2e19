"""Ends that break the rule of expert_mm: what they count as, in every kernel."""

import pytest
import torch

import adambridge_amd as ab

pytestmark = pytest.mark.gpu


# streamed, small, large and FP32 tiles, sizes below a piece; sums in parts; more experts than a wavefront has lanes
@pytest.mark.parametrize("rows,experts,n,k,dtype", [
    (40, 7, 48, 96, torch.bfloat16), (300, 7, 512, 2048, torch.bfloat16), (5000, 4, 1024, 2048, torch.bfloat16),
    (3000, 150, 136, 72, torch.bfloat16), (900, 7, 129, 77, torch.bfloat16), (40, 7, 48, 96, torch.float32),
    (2000, 130, 100, 60, torch.float32), (5000, 3, 200, 70, torch.float32), (700, 9, 5, 3, torch.bfloat16), (700, 9, 3, 90, torch.float32)])
def test_ends_below_one_before_them(rows, experts, n, k, dtype):
    gen = torch.Generator("cuda").manual_seed(rows)
    x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(experts, n, k, generator=gen, device="cuda").to(dtype).requires_grad_()
    g = torch.randn(rows, n, generator=gen, device="cuda").to(dtype)
    sorted_ends = torch.linspace(rows // 9, rows - rows // 9, experts, device="cuda")
    noise = torch.randint(-rows // 4, rows // 4, (experts,), generator=gen, device="cuda")
    one_low = sorted_ends.clone()
    one_low[experts // 2] = -5
    for ends in (sorted_ends + noise, one_low, sorted_ends.flip(0), torch.full_like(sorted_ends, rows + 9)):
        ends = ends.int()
        results = []
        for e in (ends, ends.clamp(0, rows).cummax(0).values.int()):
            out = ab.expert_mm(x, w, e)
            results.append((out, *torch.autograd.grad(out, (x, w), g)))
        assert all(torch.equal(a, b) for a, b in zip(*results))
