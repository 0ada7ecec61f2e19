"""expert_mlp's two kernels against the definition in 64 bits, and what a call of more tokens, or a trained one, takes."""

import pytest
import torch
import torch.nn.functional as F

import adambridge_amd as ab
from adambridge_amd import _hip

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _operands(tokens, experts, inter, hidden, dtype, gated, gen, logits_dtype=FP32):
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype)
    logits = torch.randn(tokens, experts, generator=gen, device="cuda").to(logits_dtype)
    up, gate, down = (torch.randn(*s, generator=gen, device="cuda").mul_(s[2] ** -0.5).to(dtype)
                      for s in ((experts, inter, hidden), (experts, inter, hidden), (experts, hidden, inter)))
    return x, logits, up, down, gate if gated else None


def _definition(x, logits, up, down, top_k, gate, activation, normalize):
    """The result in 64 bits, and a bound of the kernels' error: FP32 sums of n terms are off by n U of the terms' sizes, an
    activation, whose slope is below 1.2, by that of its operand and 16 U of the operand's size, then rounded to the type; a weight by
    2^-17 of itself."""
    eps = torch.finfo(x.dtype).eps / 2
    act = {"gelu": F.gelu, "silu": F.silu}[activation]
    x, logits, up, down = x.double(), logits.double(), up.double(), down.double()
    inter, hidden = up.shape[1:]
    out, bound = torch.zeros_like(x), torch.zeros_like(x)
    weights, chosen = torch.sort(logits, dim=1, descending=True, stable=True)
    chosen = chosen[:, :top_k]
    p = torch.softmax(weights[:, :top_k], 1) if normalize else torch.softmax(weights, 1)[:, :top_k]
    for t in range(x.shape[0]):
        for j in range(top_k):
            e = chosen[t, j]
            u, wrong_u = up[e] @ x[t], (hidden + 1) * U * (up[e].abs() @ x[t].abs())
            if gate is None:
                a, wrong = act(u), 1.2 * wrong_u + 16 * U * u.abs()
            else:
                g, wrong_g = gate[e].double() @ x[t], (hidden + 1) * U * (gate[e].double().abs() @ x[t].abs())
                a = act(g) * u
                wrong = (1.2 * wrong_g + 16 * U * g.abs()) * (u.abs() + wrong_u) + act(g).abs() * wrong_u + U * a.abs()
            wrong = wrong + eps * (a.abs() + wrong)
            out[t] += p[t, j] * (down[e] @ a)
            size = down[e].abs() @ (a.abs() + wrong)
            bound[t] += p[t, j] * (down[e].abs() @ wrong + (inter + top_k + 20) * U * size + 2.0 ** -17 * size)
    return out, bound + out.abs() * eps


def _check(tokens, experts, top_k, inter, hidden, dtype, gated, activation, normalize, gen, logits_dtype=FP32):
    x, logits, up, down, gate = _operands(tokens, experts, inter, hidden, dtype, gated, gen, logits_dtype)
    got = ab.expert_mlp(x, logits, up, down, top_k, gate, activation, normalize)
    want, bound = _definition(x, logits, up, down, top_k, gate, activation, normalize)
    assert got.dtype == dtype and got.shape == x.shape and ((got.double() - want).abs() <= bound).all()
    assert torch.equal(ab.expert_mlp(x, logits, up, down, top_k, gate, activation, normalize), got)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tokens,experts,top_k,inter,hidden", [
    (1, 1, 1, 1, 1), (1, 1, 1, 8, 8), (1, 8, 2, 16, 32), (2, 3, 3, 17, 9), (3, 64, 8, 96, 264), (5, 5, 2, 193, 333), (7, 65, 5, 40, 100),
    (16, 64, 8, 24, 40), (16, 256, 3, 33, 64), (9, 257, 64, 8, 24), (16, 1024, 64, 9, 17), (4, 200, 1, 300, 40), (1, 64, 6, 2056, 520),
    (13, 4, 2, 520, 2050), (16, 2, 1, 4099, 72), (11, 6, 6, 1000, 24)])
@pytest.mark.parametrize("gated,activation,normalize", [(False, "gelu", True), (True, "silu", False)])
def test_the_layer(tokens, experts, top_k, inter, hidden, gated, activation, normalize, dtype):
    gen = torch.Generator("cuda").manual_seed(tokens * experts + inter)
    _check(tokens, experts, top_k, inter, hidden, dtype, gated, activation, normalize, gen)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_variants(dtype):
    gen = torch.Generator("cuda").manual_seed(0)
    for gated in (False, True):
        for activation in ("gelu", "silu"):
            for normalize in (False, True):
                for logits_dtype in (BF16, FP32):
                    _check(6, 12, 3, 72, 48, dtype, gated, activation, normalize, gen, logits_dtype)


def test_the_kernels_and_the_operators_choose_alike():
    """Equal logits, masked ones, NaN; a token without any logit above -inf has a result of zeros."""
    gen = torch.Generator("cuda").manual_seed(1)
    x, logits, up, down, _ = _operands(8, 70, 24, 40, FP32, False, gen)
    logits = logits.mul(2).round()   # many equal
    logits[1] = -torch.inf
    logits[2, :66] = -torch.inf
    logits[3, 5] = torch.nan
    logits[4] = 0.0
    logits[4, ::2] = -0.0
    for normalize in (True, False):
        got = ab.expert_mlp(x, logits, up, down, 6, normalize=normalize)
        r = ab.route(logits, 6, normalize)
        want = ab.combine(ab.expert_mm(F.gelu(ab.expert_mm(ab.dispatch(x, r), up, r.ends)), down, r.ends), r)
        assert torch.allclose(got, want, rtol=1e-4, atol=1e-5, equal_nan=True)
        assert not got[1].any() and got[3].isnan().all() and got[[0, 2, 4, 5, 6, 7]].isfinite().all()


def test_what_an_expert_holds_stays_with_its_tokens():
    gen = torch.Generator("cuda").manual_seed(2)
    for dtype in (BF16, FP32):
        for sizes in ((24, 40), (33, 41)):
            x, logits, up, down, gate = _operands(10, 6, *sizes, dtype, True, gen)
            clean = ab.expert_mlp(x, logits, up, down, 2, gate)
            chose = (ab.route(logits, 2).experts == 3).any(1)
            assert 0 < chose.sum() < 10
            for poisoned in (up, gate, down):
                kept = poisoned[3].clone()
                poisoned[3] = torch.nan
                got = ab.expert_mlp(x, logits, up, down, 2, gate)
                assert torch.equal(got[~chose], clean[~chose]) and got[chose].isnan().all()
                poisoned[3] = kept
            x[4] = torch.inf
            got = ab.expert_mlp(x, logits, up, down, 2, gate)
            others = torch.arange(10, device="cuda") != 4
            assert torch.equal(got[others], clean[others])


def test_more_tokens_and_gradients_take_the_operators(monkeypatch):
    gen = torch.Generator("cuda").manual_seed(3)
    x, logits, up, down, gate = _operands(17, 6, 40, 24, FP32, True, gen)
    few = torch.cat([ab.expert_mlp(x[i:i + 9], logits[i:i + 9], up, down, 2, gate, "silu") for i in (0, 9)])
    assert torch.allclose(ab.expert_mlp(x, logits, up, down, 2, gate, "silu"), few, rtol=1e-4, atol=1e-5)
    leaves = [t.clone().requires_grad_() for t in (x[:5], logits[:5], up, down, gate)]
    y = ab.expert_mlp(*leaves[:4], 2, leaves[4], "silu")
    assert torch.allclose(y, few[:5], rtol=1e-4, atol=1e-5)
    g = torch.randn(5, 24, generator=gen, device="cuda")
    got = torch.autograd.grad(y, leaves, g)
    there = [t.detach().cpu().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(ab.expert_mlp(*there[:4], 2, there[4], "silu"), there, g.cpu().double())
    for a, b in zip(got, want):
        assert torch.allclose(a.cpu().double(), b, rtol=1e-3, atol=1e-4)
    with torch.no_grad():
        assert torch.equal(ab.expert_mlp(*leaves[:4], 2, leaves[4], "silu"), few[:5])


def test_orders_and_alignments():
    gen = torch.Generator("cuda").manual_seed(4)
    x, logits, up, down, gate = _operands(7, 6, 40, 24, BF16, True, gen)
    want = ab.expert_mlp(x, logits, up, down, 2, gate)
    strided = [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (x, logits, up, down, gate)]
    assert torch.equal(ab.expert_mlp(*strided[:4], 2, strided[4]), want)

    def shifted(t):   # the same values off the 16-byte boundaries
        buffer = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        buffer[1:] = t.reshape(-1)
        return buffer[1:].view(t.shape)

    for moved in ((x,), (up,), (gate,), (down,), (x, up, down, gate)):
        args = [shifted(t) if any(t is m for m in moved) else t for t in (x, logits, up, down, gate)]
        got = ab.expert_mlp(*args[:4], 2, args[4])
        assert torch.allclose(got, want, rtol=2.0 ** -7, atol=2.0 ** -9)
    with torch.autocast("cuda", dtype=BF16):
        assert torch.allclose(ab.expert_mlp(x.float(), logits, up.float(), down.float(), 2, gate.float()), want, rtol=0.05, atol=0.02)


def test_between_guards():
    """Operands inside NaN, the result and the scratch inside marks."""
    lib = _hip.load()
    gen = torch.Generator("cuda").manual_seed(5)
    for dtype in (BF16, FP32):
        for inter, hidden, shift in ((24, 40, 0), (33, 41, 1), (24, 41, 3)):
            operands = _operands(9, 5, inter, hidden, dtype, True, gen)
            want = ab.expert_mlp(*operands[:4], 2, operands[4], "silu")

            def inside(t, guard):
                whole = torch.full((t.numel() + 8192,), guard, dtype=t.dtype, device="cuda")
                part = whole[4096 + shift:4096 + shift + t.numel()].view(t.shape)
                part.copy_(t)
                return whole, part

            parts = [inside(t, torch.nan)[1] for t in operands]
            whole, out = inside(torch.zeros_like(want), 777.0)
            code = {BF16: _hip.DT_BF16, FP32: _hip.DT_F32}[dtype]
            nbytes = lib._lib.adambridge_expert_mlp_work(code, 9, 5, 2, inter, hidden)
            scratch = torch.full((nbytes + 8192,), 7, dtype=torch.uint8, device="cuda")
            lib.set_stream(torch.cuda.current_stream())
            rc = lib._lib.adambridge_expert_mlp(parts[0].data_ptr(), parts[1].data_ptr(), _hip.DT_F32, parts[2].data_ptr(), parts[4].data_ptr(),
                                                parts[3].data_ptr(), code, 9, 5, 2, inter, hidden, 1, 1, out.data_ptr(), scratch.data_ptr() + 4096)
            assert rc == 0
            assert torch.allclose(out, want, rtol=2.0 ** -7 if dtype == BF16 else 1e-4, atol=2.0 ** -9 if dtype == BF16 else 1e-5)
            assert (scratch[:4096] == 7).all() and (scratch[4096 + nbytes:] == 7).all()
            assert (whole[:4096 + shift] == 777).all() and (whole[4096 + shift + out.numel():] == 777).all()


def test_replayed_from_a_graph():
    """With other logits and rows at each replay, and eager calls between."""
    gen = torch.Generator("cuda").manual_seed(6)
    x, logits, up, down, _ = _operands(4, 64, 72, 48, BF16, False, gen)
    ab.expert_mlp(x, logits, up, down, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ab.expert_mlp(x, logits, up, down, 4)
    for _ in range(4):
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        logits.copy_(torch.randn(logits.shape, generator=gen, device="cuda"))
        graph.replay()
        want = ab.expert_mlp(x, logits, up, down, 4)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
