"""Calls of embed, token_losses and expert_mlp that are not the ordinary ones: what reaches a kernel, and what must not; and the
operators together, as a model's training step and its decoding use them."""

import threading

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn.functional as F

import adambridge_amd as ab
from adambridge_amd import _hip, experts, vocabulary

pytestmark = pytest.mark.gpu

NAMES = ("embed", "token_losses", "token_losses_few")


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _operator(name, dtype=torch.float32, gen=None):
    """The operator as a function of its differentiable operands, and those."""
    gen = gen or _gen(len(name))
    leaf = lambda *shape: torch.randn(*shape, generator=gen, device="cuda").to(dtype).requires_grad_()
    if name == "embed":
        ids = torch.randint(0, 24, (5, 14), generator=gen, device="cuda")
        return lambda w: ab.embed(ids.to(w.device), w, 1.5, 3), [leaf(24, 40)]
    rows = 70 if name == "token_losses" else 9
    t = torch.randint(0, 30, (rows,), generator=gen, device="cuda")
    t[::4] = -100
    return lambda h, w: ab.token_losses(h, w, t.to(w.device)), [leaf(rows, 40), leaf(30, 40)]


def _gradients(name, dtype=torch.float32, seed=1):
    fn, leaves = _operator(name, dtype)
    out = fn(*leaves)
    g = torch.randn(out.shape, generator=_gen(seed), device="cuda").to(out.dtype)
    return torch.autograd.grad(out, leaves, g)


def _near(got, want):
    return torch.allclose(got, want, rtol=1e-4, atol=1e-5 * (1.0 + want.abs().max().item()))


def _mlp():
    gen = _gen(5)
    return [torch.randn(*s, generator=gen, device="cuda") * 0.3 for s in ((9, 40), (9, 6), (6, 24, 40), (6, 40, 24))]


# ------------------------------------------------------- differentiated in other ways

@pytest.mark.parametrize("name", NAMES)
def test_a_gradient_s_tangent_is_carried_on(name):
    """Forward mode over a backward pass whose incoming gradient is dual: the gradient is linear in it."""
    fn, leaves = _operator(name)
    out = fn(*leaves)
    scale, tangent = (torch.randn(out.shape, generator=_gen(s), device="cuda") for s in (5, 6))
    with forward_ad.dual_level():
        grads = torch.autograd.grad((fn(*leaves) * forward_ad.make_dual(scale, tangent)).sum(), leaves)
        got = [forward_ad.unpack_dual(t) for t in grads]
        got = [(t.primal.clone(), None if t.tangent is None else t.tangent.clone()) for t in got]
    want = zip(torch.autograd.grad(out, leaves, scale, retain_graph=True), torch.autograd.grad(out, leaves, tangent))
    for (primal, moved), (want_primal, want_moved) in zip(got, want):
        assert moved is not None and _near(primal, want_primal) and _near(moved, want_moved)


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives(name):
    """As torch operations differentiate the definition in 64 bits."""
    fn, leaves = _operator(name)
    results = []
    for cast in (lambda t: t, lambda t: t.cpu().double()):
        here = [cast(t.detach()).requires_grad_() for t in leaves]
        out = fn(*here)
        g, *moves = [cast(torch.randn(t.shape, generator=_gen(20 + i), device="cuda")) for i, t in enumerate((out, *here))]
        g.requires_grad_()
        first = torch.autograd.grad((out * out * g).sum(), here, create_graph=True)
        second = torch.autograd.grad(sum((a * m).sum() for a, m in zip(first, moves)), [g, *here])
        results.append([t.cpu().float() for t in second])
    for got, want in zip(*results):
        assert torch.allclose(got, want, rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_and_batched_gradients(name):
    fn, leaves = _operator(name)
    out = fn(*leaves)
    g = torch.randn(3, *out.shape, generator=_gen(1), device="cuda")
    want = torch.autograd.grad(out, leaves, g[0], retain_graph=True)
    free = [t.detach() for t in leaves]
    got = torch.func.grad(lambda *ts: (fn(*ts) * g[0]).sum(), argnums=tuple(range(len(free))))(*free)
    assert all(_near(a, b) for a, b in zip(got, want))
    moves = [torch.randn(t.shape, generator=_gen(8 + i), device="cuda") for i, t in enumerate(free)]
    primal, moved = torch.func.jvp(fn, tuple(free), tuple(moves))
    assert _near(primal, out.detach())
    assert torch.allclose((moved * g[0]).sum(), sum((a * b).sum() for a, b in zip(want, moves)), rtol=1e-3, atol=1e-2)
    twice = torch.func.vmap(fn, in_dims=(0,) + (None,) * (len(free) - 1))(torch.stack((free[0], 2 * free[0])), *free[1:])
    assert _near(twice[0], out.detach()) and _near(twice[1], fn(2 * free[0], *free[1:]))
    at_once = torch.autograd.grad(out, leaves, g, is_grads_batched=True)
    for i in range(3):
        one = torch.autograd.grad(fn(*leaves), leaves, g[i])
        assert all(torch.allclose(a[i], b, rtol=1e-3, atol=1e-4) for a, b in zip(at_once, one))


def test_gradients_against_differences():
    """embed is linear in its weight; token_losses' slope along a direction is its gradient's part along it."""
    fn, (w,) = _operator("embed")
    d, g = torch.randn(w.shape, generator=_gen(1), device="cuda"), torch.randn(5, 14, 40, generator=_gen(2), device="cuda")
    grad, = torch.autograd.grad(fn(w), w, g)
    with torch.no_grad():
        moved = torch.where((torch.arange(24, device="cuda") == 3)[:, None], 0.0, d)   # the padding has no gradient
        want = ((fn(w + moved) - fn(w - moved)).double() * g.double()).sum() / 2
    assert abs(want - (grad.double() * d.double()).sum()) <= 2800 ** 0.5 * 16 * 2.0 ** -22
    for name in NAMES[1:]:
        fn, leaves = _operator(name)
        g = torch.rand(leaves[0].shape[0], generator=_gen(3), device="cuda")
        grads = torch.autograd.grad(fn(*leaves), leaves, g)
        with torch.no_grad():
            for i in range(2):
                d = torch.randn(leaves[i].shape, generator=_gen(4), device="cuda")
                step = 2.0 ** -7
                up, down = (fn(*[t + s * step * d if j == i else t for j, t in enumerate(leaves)]).double() for s in (1, -1))
                want = ((up - down) * g.double()).sum() / (2 * step)
                # curvature: a third of a step squared times the logits' moves, up to 40, cubed, over 70 rows; rounding: 2^-18 a loss over a step
                assert abs(want - (grads[i].double() * d.double()).sum()) <= 70 * (step ** 2 * 40.0 ** 3 / 6 + 2.0 ** -17 / step)


# ------------------------------------------------------------------------- saved tensors

def _strided(t):
    return torch.stack((t, t), 1)[:, 0] if t.dim() == 1 else t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_that_come_back_strided(name, dtype):
    want = _gradients(name, dtype)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _strided):
        got = _gradients(name, dtype)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES[1:])
def test_saved_tensors_that_come_back_of_another_type(name):
    want = _gradients(name)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.double() if t.is_floating_point() else t):
        got = _gradients(name)
    assert all(_near(a.float(), b) for a, b in zip(got, want))


@pytest.mark.parametrize("back", [lambda t: t[:-1], lambda t: t[..., None], lambda t: t.cpu()],
                         ids=["fewer", "another dimension", "the host's"])
@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_that_cannot_be_the_operand_s_are_refused(name, back):
    for create_graph in (False, True):
        fn, leaves = _operator(name)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back), pytest.raises(RuntimeError, match="came back|same device"):
            out = fn(*leaves)
            torch.autograd.grad(out, leaves, torch.ones_like(out), create_graph=create_graph)


def test_a_weight_written_in_place_is_refused():
    fn, (h, w) = _operator("token_losses")
    loss = fn(h, w).sum()
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# --------------------------------------------------------------- modes, threads, refusals

def test_a_default_device_leaves_the_kernels_on(monkeypatch):
    want, mlp = [_gradients(name) for name in NAMES], ab.expert_mlp(*_mlp(), 2)
    for module, name in ((vocabulary, "_torch_embed"), (vocabulary, "_torch_token_losses"), (experts, "route")):
        monkeypatch.setattr(module, name, None)
    for device in ("cuda", "cpu"):
        with torch.device(device):
            got, out = [_gradients(name) for name in NAMES], ab.expert_mlp(*_mlp(), 2)
        assert all(torch.equal(a, b) for one, two in zip(got, want) for a, b in zip(one, two)) and torch.equal(out, mlp)


def test_a_mode_that_observes_operations_sees_them():
    class Count(torch.overrides.TorchFunctionMode):
        def __init__(self):
            self.seen = 0

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.seen += 1
            return func(*args, **(kwargs or {}))

    for call in [lambda n=n: _operator(n)[0](*_operator(n)[1]) for n in NAMES] + [lambda: ab.expert_mlp(*_mlp(), 2)]:
        with Count() as count:
            call()
        assert count.seen > 8


def test_compiled_calls():
    """Outside the graph, with the same values."""
    for name in NAMES:
        fn, leaves = _operator(name)
        assert torch.equal(torch.compile(fn, backend="eager")(*leaves), fn(*leaves))
    args = _mlp()
    assert torch.equal(torch.compile(lambda *a: ab.expert_mlp(*a, 2) * 1.0, backend="eager")(*args), ab.expert_mlp(*args, 2))


def test_tensors_without_memory_take_torch_operations():
    zero = lambda *shape: torch._efficientzerotensor(shape, device="cuda")
    ids = torch.tensor([1, 2], device="cuda")
    assert not ab.embed(ids, zero(5, 8)).any()
    assert torch.allclose(ab.token_losses(zero(2, 8), torch.randn(5, 8, device="cuda"), ids), torch.full((2,), 5.0, device="cuda").log())
    x, logits, up, down = _mlp()
    assert not ab.expert_mlp(zero(9, 40), logits, up, down, 2).any()


def test_threads_have_a_stream_each():
    want, mlp = [_gradients(name) for name in NAMES], ab.expert_mlp(*_mlp(), 2)
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = [_gradients(name) for name in NAMES], ab.expert_mlp(*_mlp(), 2)
                torch.cuda.current_stream().synchronize()
        except Exception as error:   # reported by the thread that asserts
            errors.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors and len(got) == 3
    for one, out in got.values():
        assert all(torch.equal(a, b) for x, y in zip(one, want) for a, b in zip(x, y)) and torch.equal(out, mlp)


def test_calls_that_are_not_ordinary_ones_are_left_to_python():
    """The native calls answer None, before anything is done, to what their kernels do not take."""
    o = _hip.ops()
    ids, w, h = torch.tensor([1, 2], device="cuda"), torch.randn(5, 8, device="cuda"), torch.randn(2, 8, device="cuda")
    for args in ((ids.cpu(), w, 1.0, None), (ids.short(), w, 1.0, None), (ids.float(), w, 1.0, None), (ids, w.half(), 1.0, None),
                 (ids, w.t(), 1.0, None), (ids, w[0], 1.0, None), (ids, w[:0], 1.0, None), (ids, w, 1, None), (ids, w, 1.0, 5), (ids, w, 1.0, -1),
                 (ids, w, 1.0, True), (ids, w, 1.0, 1 << 70), (ids[:0], w, 1.0, None), (torch.stack((ids, ids), 1)[:, 0], w, 1.0, None),
                 ([1, 2], w, 1.0, None), (ids, w, 1.0)):
        assert o.embed(*args) is None
    for args in ((h.cpu(), w, ids, -100), (h, w.bfloat16(), ids, -100), (h.half(), w.half(), ids, -100), (h, w, ids.int(), -100),
                 (h, w, ids[:1], -100), (h, w[:, :4], ids, -100), (h[:, :4], w, ids, -100), (h, w, ids, 1.0), (h, w, ids, True), (h, w, ids, 1 << 70),
                 (h[:0], w, ids[:0], -100), (h[:, :3].contiguous(), w[:, :3].contiguous(), ids, -100), (h.t(), w, ids, -100),
                 (h, w, ids.cpu(), -100), (h, w, None, -100)):
        assert o.token_losses(*args) is None
    x, logits, up, down = _mlp()
    for args in ((x, logits, up, down, None, 2, False, 1), (x, logits, up, down, None, 7, False, True), (x, logits, up, down, None, 0, False, True),
                 (x, logits, up, down, None, True, False, True), (x, logits, up, down, down, 2, False, True),
                 (x.bfloat16(), logits, up, down, None, 2, False, True), (x, logits.half(), up, down, None, 2, False, True),
                 (x, logits[:8], up, down, None, 2, False, True), (x, logits[:, :5].contiguous(), up, down, None, 2, False, True),
                 (x, logits, up, up, None, 2, False, True), (x[:0], logits[:0], up, down, None, 2, False, True),
                 (torch.cat((x, x)), torch.cat((logits, logits)), up, down, None, 2, False, True),
                 (x.clone().requires_grad_(), logits, up, down, None, 2, False, True), (x, logits, up, down, None, 2, False)):
        assert o.expert_mlp(*args) is None
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert o.token_losses(h, w, ids, -100) is None and o.expert_mlp(x, logits, up, down, None, 2, False, True) is None
    with pytest.raises(ValueError, match="ids must be int64 or int32 on cuda"):
        ab.embed(ids.cpu(), w)
    with pytest.raises(ValueError, match="on one device"):
        ab.token_losses(h, w, ids.cpu())
    with pytest.raises(ValueError, match="on one device"):
        ab.expert_mlp(x, logits.cpu(), up, down, 2)
    assert ab.embed(ids, w.half()).dtype == torch.float16   # torch operations
    assert ab.token_losses(h.double(), w.double(), ids).dtype == torch.float64


# ------------------------------------------------------------------------------- together

def _model(dtype=torch.bfloat16, vocab=200, hidden=64, inter=96, n=6):
    gen = _gen(7)
    rand = lambda *s: (torch.randn(*s, generator=gen, device="cuda") * s[-1] ** -0.5).to(dtype).requires_grad_()
    return dict(embed=rand(vocab, hidden), norm=torch.ones(hidden, device="cuda", dtype=dtype, requires_grad=True), router=rand(n, hidden),
                up=rand(n, inter, hidden), gate=rand(n, inter, hidden), down=rand(n, hidden, inter))


def _losses(p, ids, targets, head="embed"):
    x = ab.embed(ids, p["embed"], 8.0, padding_idx=0)
    flat = x.reshape(-1, x.shape[-1])
    h = ab.layer_norm(flat, p["norm"])
    flat = flat + ab.expert_mlp(h, h @ p["router"].t(), p["up"], p["down"], 2, p["gate"], "silu")
    return ab.token_losses(flat.reshape(x.shape), p[head], targets)


def test_a_model_of_the_operators_trains_with_a_tied_embedding():
    """Losses and gradients against the same model in 64 bits on the CPU; the embedding has those of both its uses."""
    p = _model(torch.float32)
    ids = torch.randint(0, 200, (3, 40), generator=_gen(8), device="cuda")
    ids[1, 20:] = 0
    targets = torch.where(ids == 0, -100, ids.roll(-1, 1))
    loss = _losses(p, ids, targets)
    got = torch.autograd.grad(loss.sum(), list(p.values()))
    there = {k: v.detach().cpu().double().requires_grad_() for k, v in p.items()}
    x = F.embedding(ids.cpu(), there["embed"], 0) * 8.0
    flat = x.reshape(-1, 64)
    h = F.layer_norm(flat, (64,), there["norm"])
    weights, chosen = torch.topk(h @ there["router"].t(), 2)
    weights = torch.softmax(weights, 1)
    moved = []
    for t in range(len(flat)):
        moved.append(sum(w * (there["down"][e] @ (F.silu(there["gate"][e] @ h[t]) * (there["up"][e] @ h[t]))) for w, e in zip(weights[t], chosen[t])))
    want = F.cross_entropy((flat + torch.stack(moved)) @ there["embed"].t(), targets.cpu().reshape(-1), reduction="none").view(3, 40)
    assert torch.allclose(loss.detach().cpu().double(), want, rtol=1e-4, atol=1e-4)
    for a, b in zip(got, torch.autograd.grad(want.sum(), list(there.values()))):
        assert torch.allclose(a.cpu().double(), b, rtol=1e-3, atol=1e-3 * b.abs().max().item())


def test_a_training_step_captured_in_a_graph():
    """Replayed with other tokens, eager steps between: every replay gives the eager step's values."""
    p = _model()
    ids = torch.randint(1, 200, (4, 100), generator=_gen(9), device="cuda")
    targets = ids.roll(-1, 1).contiguous()
    seed = torch.rand(4, 100, generator=_gen(10), device="cuda")

    def once():
        loss = _losses(p, ids, targets)
        return (loss.detach(), *torch.autograd.grad(loss, list(p.values()), seed))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once()
    for i in range(4):
        ids.copy_(torch.randint(0, 200, ids.shape, generator=_gen(30 + i), device="cuda"))
        targets.copy_(torch.where(ids < 50 * i, -100, ids.roll(-1, 1)))   # another number of scored rows each time
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, once())), i


def test_two_graphs_replayed_in_turn():
    """Each has its own scratch."""
    p = _model()
    ids = [torch.randint(1, 200, (1, n), generator=_gen(n), device="cuda") for n in (7, 90)]

    def once(i):
        with torch.no_grad():
            return _losses(p, ids[i], ids[i].roll(-1, 1))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [once(0).clone(), once(1).clone()]
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(once(i))
    for _ in range(3):
        for i in (0, 1, 1, 0):
            outs[i].zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])


def test_on_another_stream():
    p = _model()
    ids = torch.randint(0, 200, (2, 60), generator=_gen(11), device="cuda")
    targets = torch.where(ids == 0, -100, ids.roll(-1, 1))
    want = torch.autograd.grad(_losses(p, ids, targets).sum(), list(p.values()))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            got = torch.autograd.grad(_losses(p, ids, targets).sum(), list(p.values()))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_decoding_step_is_the_whole_sequence_s_last_row():
    """Up to 16 sequences one token at a time, by the kernels for few tokens, against the operators of the whole batch."""
    p = {k: v.detach() for k, v in _model(torch.float32).items()}
    ids = torch.randint(1, 200, (16, 12), generator=_gen(12), device="cuda")
    whole = _losses(p, ids, ids.roll(-1, 1))
    for t in range(12):
        assert torch.allclose(_losses(p, ids[:, t], ids.roll(-1, 1)[:, t]), whole[:, t], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,size", [(51, 74, 2056), (700, 300, 1030), (16, 500, 1544), (1100, 4099, 2056)])
def test_sums_in_parts_captured_in_a_graph(rows, vocab, size, dtype):
    """Few tiles, whose sums are cut and joined: replayed with other targets, after scratch of NaN, as the eager calls."""
    gen = _gen(rows)
    h = torch.randn(rows, size, generator=gen, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(vocab, size, generator=gen, device="cuda") * size ** -0.5).to(dtype).requires_grad_()
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    seed = torch.rand(rows, generator=gen, device="cuda")

    def once():
        y = ab.token_losses(h, w, t)
        table = ab.embed(t[:200], w)
        return (y.detach(), *torch.autograd.grad(y, (h, w), seed), *torch.autograd.grad(table, w, h[:200].detach()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once()
    for i in range(4):
        t.copy_(torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.3 * i, -100, torch.randint(0, vocab, (rows,), generator=gen, device="cuda")))
        graph.replay()
        torch.cuda.synchronize()
        torch.full((1 << 26,), torch.nan, device="cuda")
        eager = once()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), i
        assert not any(x.isnan().any() for x in eager)
